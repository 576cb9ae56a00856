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

template <class T, int NT>
__global__ __launch_bounds__(NT) void quantize_rows_kernel(const T* __restrict__ x, signed char* __restrict__ q,
                                                           float* __restrict__ scale, int K, int ldq) {
  constexpr int VEC = gmk_elem<T>::VEC;
  __shared__ float red[2 * NT / 64];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * K;
  float mx = 0.f, bad = 0.f;
  for (int e = threadIdx.x * VEC; e < K; e += NT * VEC) gmk_quantize_scan<T>(gmk_row_piece(xr, e, K), K - e, mx, bad);
  mx = gmk_block_max_all<NT>(mx, red);
  bad = gmk_block_max_all<NT>(bad, red);
  const float s = gmk_quantize_scale(mx);
  const float inv = bad == 0.f ? 1.0f / s : 0.f;
  for (int e = threadIdx.x * VEC; e < ldq; e += NT * VEC) {
    unsigned w[2] = {0u, 0u};
    if (e < K) gmk_quantize_piece<T>(gmk_row_piece(xr, e, K), K - e, s, inv, w);
    __builtin_memcpy(q + row * ldq + e, w, VEC);
  }
  if (threadIdx.x == 0) scale[row] = bad == 0.f ? s : __builtin_nanf("");
}

int gmk_quantize_rows_launch(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq,
                             gmk_stream_t stream) {
  gmk_with_dtype(xtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((quantize_rows_kernel<T, 256>), dim3((unsigned)M), dim3(256), 0, (hipStream_t)stream, (const T*)x, q,
                       scale, K, ldq);
    return 0;
  });
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}

extern "C" int gmk_quantize_rows(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq,
                                 gmk_stream_t stream) {
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(M >= 0 && M <= GMK_MAX_ROWS && K > 0 && ldq >= K && ldq % 16 == 0, GMK_E_SHAPE);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(x && q && scale, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned16(q) && gmk_aligned_to(scale, 4), GMK_E_ALIGN);
  GMK_PLAN_HOOK(gmk_quantize_rows, x, xtype, q, scale, M, K, ldq, stream);
  return gmk_quantize_rows_launch(x, xtype, q, scale, M, K, ldq, stream);
}
