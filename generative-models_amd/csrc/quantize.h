// quantize.h -- the row quantiser's arithmetic (quantize.hip says why GmkQuant::one is exact) and its launch, for the 8-bit GEMM.
#pragma once
#include "rows.h"

// The largest magnitude of a row, as the bits of the type without their sign: their order as whole numbers is that of the magnitudes,
// infinities and NaNs above all.  16-bit types two at a time.
template <class T>
struct GmkMagnitude {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  unsigned mx = 0;
  __device__ __forceinline__ void scan(const gmk_u32x4& v) {   // the row's missing elements are zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        mx = max(mx, v[i] & 0x7FFFFFFFu);
      } else {
        const unsigned w = v[i] & 0x7FFF7FFFu;
        mx = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, mx), __builtin_bit_cast(u16x2, w)));
      }
    }
  }
  // +inf where the row holds an infinity or a NaN
  __device__ __forceinline__ float value() const {
    unsigned m = mx;
    if constexpr (sizeof(T) == 2) m = max(m & 0xFFFFu, m >> 16);
    if constexpr (std::is_same<T, __bf16>::value) m <<= 16;
    if constexpr (std::is_same<T, _Float16>::value) return m >= 0x7C00u ? __builtin_inff() : (float)__builtin_bit_cast(_Float16, (unsigned short)m);
    return __builtin_bit_cast(float, min(m, 0x7F800000u));
  }
};

// What a row's largest magnitude makes of it: its scale (NaN: the row holds an infinity or a NaN, and every q is 0) and 1 / scale.
struct GmkQuant {
  float s, inv;
  bool bad;
  __device__ __forceinline__ explicit GmkQuant(float mx) {
    bad = mx == __builtin_inff();
    s = fmaxf(mx / 127.0f, 0x1p-126f);
    inv = 1.0f / s;
  }
  __device__ __forceinline__ float scale() const { return bad ? __builtin_nanf("") : s; }
  // exact for every x
  __device__ __forceinline__ unsigned one(float x) const {
    const float q0 = rintf(x * inv);
    const float r = fmaf(-q0, s, x), h = 0.5f * s;
    int q = (int)q0;
    if (fabsf(r) > h || (fabsf(r) == h && (q & 1))) q += r > 0.f ? 1 : -1;
    return (unsigned)q & 0xFFu;
  }
  // A piece of VEC values -> VEC bytes in w[0 .. VEC / 4).  x / s is known to 127 * 2^-23 < 2e-5 from x * inv, so that only quotients that
  // close to a half need one(): a few pieces in a thousand.  Adding 1.5 * 2^23 rounds to a whole number and leaves it in the sum's low bits.
  template <class T>
  __device__ __forceinline__ void piece(const gmk_u32x4& v, unsigned* w) const {
    constexpr int VEC = gmk_elem<T>::VEC;
    const float magic = 12582912.0f;
    float u[VEC], far = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = gmk_piece<T>(v, i);
      u[i] = fmaf(x, inv, magic);
      far = fmaxf(far, fabsf(fmaf(x, inv, magic - u[i])));
    }
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      unsigned b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(unsigned, u[4 * j + i]);
      w[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400), __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400), 0x05040100);
    }
    if (far > 0.4999f || bad) {
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) {
        unsigned b = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) b |= bad ? 0u : one(gmk_piece<T>(v, 4 * j + i)) << (8 * i);
        w[j] = b;
      }
    }
  }
};

int gmk_quantize_rows_launch(const void* x, int xtype, signed char* q, float* scale, int64_t M, int K, int ldq, bool once,
                             gmk_stream_t stream);
