// gemm_i8.hip -- y = act((xq wq^T) * xscale * wscale + bias) on the 8-bit matrix instructions (v_mfma_i32_16x16x64_i8).  No
// counterpart in the reference: the 8-bit form of its nn.Linear (models/classifiers.py:19-20) for inference.
//
// The sum is a 32-bit integer, exact for K <= 131,056 (K * 128 * 128 < 2^31), so neither the order of K nor a split of it shows
// in the result.  The weight is the instruction's first operand: its 16 rows are the result's rows, so that a lane holds 4
// consecutive outputs of one row of y and stores them together.
#include "rows.h"
#include "quantize.h"
#include "plan.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The result of 4 consecutive columns n .. n+3 of row m.  (float)acc rounds sums beyond 2^24 to 24 bits, each product and the
// sum with the bias once more: four roundings of 2^-24.
template <class T>
__device__ __forceinline__ void gemm_i8_store4(const i32x4& acc, float xs, const float* __restrict__ wscale,
                                               const float* __restrict__ bias, T* __restrict__ y, int m, int n, int N, int act) {
  float4 z, d;
  float* zp = &z.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = n + i < N;
    const float v = (float)acc[i] * xs * (in ? wscale[n + i] : 0.f);
    zp[i] = bias && in ? v + bias[n + i] : v;
  }
  GMK_WITH_ACT(act, [&](auto f) { float4 a; f(z, a, d); z = a; });
  T t[4] = {(T)z.x, (T)z.y, (T)z.z, (T)z.w};
  T* p = y + (int64_t)m * N + n;
  if (n + 4 <= N) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) p[i] = t[i];
  }
}

// 4 waves, each 32 rows of w times 32 rows of x from registers: right for every shape, and no more.
template <class T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const signed char* __restrict__ xq, const float* __restrict__ xscale,
                                                      const signed char* __restrict__ wq, const float* __restrict__ wscale,
                                                      const float* __restrict__ bias, T* __restrict__ y, int M, int K, int N,
                                                      int act) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 64 + (wave & 1) * 32, m0 = blockIdx.y * 64 + (wave >> 1) * 32;
  const int r = lane & 15, kq = (lane >> 4) * 16;
  i32x4 acc[2][2] = {};
  for (int k = kq; k - kq < K; k += 64) {
    i32x4 a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + 16 * i + r, m = m0 + 16 * i + r;
      a[i] = k < K && n < N ? *(const i32x4*)(wq + (int64_t)n * K + k) : i32x4{0, 0, 0, 0};
      b[i] = k < K && m < M ? *(const i32x4*)(xq + (int64_t)m * K + k) : i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int m = m0 + 16 * j + r;
    if (m >= M) continue;
    const float xs = xscale[m];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + 16 * i + (lane >> 4) * 4;
      if (n < N) gemm_i8_store4<T>(acc[i][j], xs, wscale, bias, y, m, n, N, act);
    }
  }
}

static int gemm_i8_check(int M, int K, int N, int ytype, int act) {
  GMK_REQUIRE(gmk_dtype_ok(ytype) && act >= GMK_ACT_NONE && act <= GMK_ACT_SIGMOID, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(M >= 0 && N > 0 && K > 0, GMK_E_SHAPE);
  GMK_REQUIRE(K <= GMK_I8_MAX_K, GMK_E_TOO_LARGE);
  return GMK_OK;
}

static int gemm_i8_launch(const signed char* xq, const float* xscale, const signed char* wq, const float* wscale,
                          const float* bias, void* y, int ytype, int M, int K, int N, int act, gmk_stream_t stream) {
  GMK_REQUIRE((M + 63) / 64 <= 65535, GMK_E_TOO_LARGE);
  gmk_with_dtype(ytype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((gemm_i8_kernel<T>), dim3((N + 63) / 64, (M + 63) / 64), dim3(256), 0, (hipStream_t)stream, xq, xscale,
                       wq, wscale, bias, (T*)y, M, K, N, act);
    return 0;
  });
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}

extern "C" size_t gmk_gemm_i8_workspace_bytes(int M, int K, int N) { return 0; }

extern "C" int gmk_gemm_i8(const signed char* xq, const float* xscale, const signed char* wq, const float* wscale,
                           const float* bias, void* y, int ytype, int M, int K, int N, int act, void* ws, size_t ws_bytes,
                           gmk_stream_t stream) {
  const int rc = gemm_i8_check(M, K, N, ytype, act);
  if (rc != GMK_OK) return rc;
  GMK_REQUIRE(K % 16 == 0, GMK_E_SHAPE);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(xq && xscale && wq && wscale && y, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned16(xq) && gmk_aligned16(wq) && gmk_aligned_to(xscale, 4) && gmk_aligned_to(wscale, 4) &&
              gmk_aligned_to(bias, 4) && gmk_aligned_to(y, gmk_dtype_size(ytype)), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_gemm_i8_workspace_bytes(M, K, N), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_gemm_i8, xq, xscale, wq, wscale, bias, y, ytype, M, K, N, act, ws, ws_bytes, stream);
  return gemm_i8_launch(xq, xscale, wq, wscale, bias, y, ytype, M, K, N, act, stream);
}

// workspace of the linear layer: the quantised rows, then their scales
static size_t linear_i8_q_bytes(int M, int K) { return (size_t)M * (size_t)((K + 15) / 16 * 16); }

extern "C" size_t gmk_linear_i8_workspace_bytes(int M, int K, int N) {
  if (M <= 0 || K <= 0 || N <= 0 || K > GMK_I8_MAX_K) return 0;
  return linear_i8_q_bytes(M, K) + ((size_t)M * 4 + 15) / 16 * 16 + gmk_gemm_i8_workspace_bytes(M, (K + 15) / 16 * 16, N);
}

extern "C" int gmk_linear_i8_fwd(const void* x, int xtype, const signed char* wq, const float* wscale, const float* bias,
                                 void* y, int ytype, int M, int K, int N, int act, void* ws, size_t ws_bytes,
                                 gmk_stream_t stream) {
  const int rc = gemm_i8_check(M, K, N, ytype, act);
  if (rc != GMK_OK) return rc;
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(x && wq && wscale && y && ws, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned16(wq) && gmk_aligned_to(wscale, 4) &&
              gmk_aligned_to(bias, 4) && gmk_aligned_to(y, gmk_dtype_size(ytype)) && gmk_aligned16(ws), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_linear_i8_workspace_bytes(M, K, N), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_linear_i8_fwd, x, xtype, wq, wscale, bias, y, ytype, M, K, N, act, ws, ws_bytes, stream);
  const int Kp = (K + 15) / 16 * 16;
  signed char* q = (signed char*)ws;
  float* s = (float*)(q + linear_i8_q_bytes(M, K));
  const int e = gmk_quantize_rows_launch(x, xtype, q, s, M, K, Kp, stream);
  if (e != GMK_OK) return e;
  return gemm_i8_launch(q, s, wq, wscale, bias, y, ytype, M, Kp, N, act, stream);
}
