// quantize.h -- the row quantiser's arithmetic (quantize.hip says why it is exact) and its launch, for the 8-bit GEMM.
#pragma once
#include "rows.h"

#define GMK_MAX_ROWS 0x7FFFFFFFll   // rows of a launch: one workgroup or wave each, at most 2^31 - 1 workgroups

// mx: the largest finite magnitude so far; bad: 1 once an infinity or a NaN was met.  `left`: elements from here to the row's end.
template <class T>
__device__ __forceinline__ void gmk_quantize_scan(const gmk_u32x4& v, int left, float& mx, float& bad) {
#pragma unroll
  for (int i = 0; i < gmk_elem<T>::VEC; ++i) {
    const float a = fabsf(gmk_piece<T>(v, i));
    if (i < left) {
      if (a < __builtin_inff()) mx = fmaxf(mx, a);
      else bad = 1.f;
    }
  }
}
__device__ __forceinline__ float gmk_quantize_scale(float mx) { return fmaxf(mx / 127.0f, 0x1p-126f); }

// one value -> its whole number; inv = 1 / s, or 0 for a row that holds infinities or NaNs (then every q is 0)
__device__ __forceinline__ int gmk_quantize_one(float x, float s, float inv) {
  const float q0 = rintf(x * inv);
  const float r = fmaf(-q0, s, x), h = 0.5f * s;
  int q = (int)q0;
  const int away = r > 0.f ? 1 : -1;
  if (inv != 0.f && (fabsf(r) > h || (fabsf(r) == h && (q & 1)))) q += away;
  return inv != 0.f ? q : 0;
}

// a piece of VEC values -> VEC bytes in w[0 .. VEC / 4)
template <class T>
__device__ __forceinline__ void gmk_quantize_piece(const gmk_u32x4& v, int left, float s, float inv, unsigned* w) {
  constexpr int VEC = gmk_elem<T>::VEC;
#pragma unroll
  for (int j = 0; j < VEC / 4; ++j) {
    unsigned b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = 4 * j + i < left ? gmk_quantize_one(gmk_piece<T>(v, 4 * j + i), s, inv) : 0;
      b |= ((unsigned)q & 0xFFu) << (8 * i);
    }
    w[j] = b;
  }
}

int gmk_quantize_rows_launch(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq,
                             gmk_stream_t stream);
