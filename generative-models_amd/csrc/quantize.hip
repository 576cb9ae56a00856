// quantize.hip -- rows in 8-bit integers with one scale each: the activations (every call) and the weights (once) of the 8-bit
// linear layer.  No counterpart in the reference.
//
//   scale = max(fl32(max |x| / 127), 2^-126),   q = round_half_even(x / scale)
//
// q is exact, as if the quotient were never rounded: q0 = rint(x * (1 / scale)) is the right whole number or its neighbour
// (|x / scale| <= 127.00001, two roundings of 2^-24 each), and the remainder r = fma(-q0, scale, x) says which.  r is exact where
// it decides: near |r| = scale / 2 both x and q0 * scale are multiples of ulp(scale) / 2 and r has fewer than 25 bits.
#include "rows.h"
#include "quantize.h"
#include "plan.h"

// NT threads a row, ROWS rows a workgroup.  A thread keeps its first KEEP pieces in registers between the maximum and the rounding: rows up
// to KEEP * NT pieces are read from memory once, longer ones read their rest again.
template <class T, int NT, int ROWS, int KEEP, bool STREAM = false>
__global__ __launch_bounds__(NT * ROWS) void quantize_rows_kernel(const T* __restrict__ x, signed char* __restrict__ q,
                                                                  float* __restrict__ scale, int64_t M, int K, int ldq) {
  constexpr int VEC = gmk_elem<T>::VEC;
  static_assert(ROWS == 1 || NT == 64, "several rows a workgroup: a wave each, without a barrier");
  __shared__ float red[NT / 64];
  const int t = threadIdx.x % NT;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
  if (row >= M) return;
  const T* xr = x + row * K;
  signed char* qr = q + row * ldq;
  GmkMagnitude<T> mag;
  gmk_u32x4 keep[KEEP];
  const int e0 = t * VEC;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (e0 + i * NT * VEC < K) keep[i] = gmk_row_piece<STREAM>(xr, e0 + i * NT * VEC, K, 0.f);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (e0 + i * NT * VEC < K) mag.scan(keep[i]);
  for (int e = e0 + KEEP * NT * VEC; e < K; e += NT * VEC) mag.scan(gmk_row_piece(xr, e, K, 0.f));
  const GmkQuant qu(gmk_block_max_all<NT>(mag.value(), red));
  auto put = [&](int e, const gmk_u32x4& v) {
    unsigned w[2] = {0u, 0u};
    if (e < K) qu.piece<T>(v, w);
    __builtin_memcpy(qr + e, w, VEC);
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (e0 + i * NT * VEC < ldq) put(e0 + i * NT * VEC, keep[i]);
  for (int e = e0 + KEEP * NT * VEC; e < ldq; e += NT * VEC) put(e, e < K ? gmk_row_piece(xr, e, K, 0.f) : gmk_u32x4{0u, 0u, 0u, 0u});
  if (t == 0) scale[row] = qu.scale();
}

// 1024 threads a row where there are too few rows to fill the card and a row has work for them; a wave a row where rows are short
// (8192x512 bf16: 5.7 us, with 256 threads 10.1); else 256 threads (8192x2048 fp32: 17.6 us, a wave a row 20.6).  Bound by memory with many
// rows (8192x4096 bf16: 21.0 us, 4.8 TB/s in and out), by latency with few (256x4096 fp32: 3.8 us, with 256 threads a row 4.3, an empty launch 2.6).
// `once`: x is read past the caches, for the sake of what the caller needs in them afterwards.
int gmk_quantize_rows_launch(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq, bool once,
                             gmk_stream_t stream) {
  return gmk_with_dtype(xtype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int VEC = gmk_elem<T>::VEC;
    auto go = [&](auto kernel, int64_t blocks, int threads) -> int {
      GMK_REQUIRE(gmk_grid_ok(blocks, threads), GMK_E_TOO_LARGE);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, (hipStream_t)stream, (const T*)x, q, scale, M, K, ldq);
      GMK_CHECK_LAUNCH();
      return GMK_OK;
    };
    if (M <= 512 && K > 256 * VEC) return go(quantize_rows_kernel<T, 1024, 1, 4>, M, 1024);
    if (K <= 128 * VEC) return go(quantize_rows_kernel<T, 64, 4, 2>, (M + 3) / 4, 256);
    if (once) return go(quantize_rows_kernel<T, 256, 1, 4, true>, M, 256);
    return go(quantize_rows_kernel<T, 256, 1, 4>, M, 256);
  });
}

extern "C" int gmk_quantize_rows(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq,
                                 gmk_stream_t stream) {
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(M >= 0 && K > 0 && ldq >= K && ldq % 16 == 0, GMK_E_SHAPE);
  GMK_REQUIRE(ldq <= 1 << 30, GMK_E_TOO_LARGE);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(x && q && scale, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned16(q) && gmk_aligned_to(scale, 4), GMK_E_ALIGN);
  GMK_PLAN_HOOK(gmk_quantize_rows, x, xtype, q, scale, M, K, ldq, stream);
  return gmk_quantize_rows_launch(x, xtype, q, scale, M, K, ldq, false, stream);
}
