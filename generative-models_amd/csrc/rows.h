// rows.h -- what the row operators (quantize.hip, topk.hip, distill.hip) and the 8-bit GEMM's epilogue share: the three
// element types, 16-byte pieces of a row, and workgroup reductions.
#pragma once
#include "gmk_common.h"

typedef unsigned gmk_u32x4 __attribute__((ext_vector_type(4)));

template <class T> struct gmk_elem;
template <> struct gmk_elem<float> { enum { VEC = 4 }; };
template <> struct gmk_elem<__bf16> { enum { VEC = 8 }; };
template <> struct gmk_elem<_Float16> { enum { VEC = 8 }; };

static inline bool gmk_dtype_ok(int t) { return t == GMK_F32 || t == GMK_BF16 || t == GMK_F16; }
static inline int gmk_dtype_size(int t) { return t == GMK_F32 ? 4 : 2; }
static inline bool gmk_aligned_to(const void* p, int size) { return (((uintptr_t)p) & (unsigned)(size - 1)) == 0; }

// A launch has fewer than 2^32 threads.
static inline bool gmk_grid_ok(int64_t blocks, int threads) { return blocks > 0 && blocks <= 0xFFFFFFFFll / threads; }

// Calls f(T()) with the C++ type of a gmk_dtype (which the caller has checked).
template <class F>
static inline auto gmk_with_dtype(int t, F&& f) {
  if (t == GMK_BF16) return f(__bf16());
  if (t == GMK_F16) return f(_Float16());
  return f(float());
}

// A 16-byte piece of a row, from any address that is aligned to the element: rows of odd lengths start anywhere, and gfx950
// reads and writes 16 bytes at any alignment.  STREAM: the piece is not worth a place in the caches.
typedef unsigned gmk_u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM = false, class T>
__device__ __forceinline__ gmk_u32x4 gmk_load16(const T* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const gmk_u32x4_at2*)p);
  gmk_u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <bool STREAM, class T>
__device__ __forceinline__ void gmk_store16(T* p, const gmk_u32x4& v) {
  if constexpr (STREAM) {
    asm volatile("");   // or the compiler makes one store of this and another branch's, without the hint
    __builtin_nontemporal_store((gmk_u32x4_at2)v, (gmk_u32x4_at2*)p);
    asm volatile("");
  } else {
    __builtin_memcpy(p, &v, 16);
  }
}

// element i (a constant) of a piece, as fp32
template <class T>
__device__ __forceinline__ float gmk_piece(const gmk_u32x4& v, int i) {
  const unsigned w = v[sizeof(T) == 4 ? i : i >> 1];   // a copy: a bit cast of a vector's element itself takes element 0
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, w);
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_bit_cast(float, (i & 1) ? (w & 0xFFFF0000u) : (w << 16));
  } else {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)((i & 1) ? (w >> 16) : w));
  }
}

// VEC fp32 values as a piece of T: the one rounding (to nearest, ties to even) of an output in 16 bits
template <class T>
__device__ __forceinline__ gmk_u32x4 gmk_pack(const float* f) {
  gmk_u32x4 v;
  if constexpr (sizeof(T) == 4) {
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, f[i]);
  } else {
    typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T2 t = {(T)f[2 * i], (T)f[2 * i + 1]};
      v[i] = __builtin_bit_cast(unsigned, t);
    }
  }
  return v;
}

// The piece of a row that starts at element e: whole pieces in one load, the last, partial one element by element, its
// missing elements `fill` (-inf leaves a maximum and a sum of exponentials as they are, 0 a largest magnitude).
template <bool STREAM = false, class T>
__device__ __forceinline__ gmk_u32x4 gmk_row_piece(const T* row, int64_t e, int64_t C, float fill = -__builtin_inff()) {
  constexpr int VEC = gmk_elem<T>::VEC;
  if (e + VEC <= C) return gmk_load16<STREAM>(row + e);
  T t[VEC];
  if (e >= C) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (T)fill;
    gmk_u32x4 v;
    __builtin_memcpy(&v, t, 16);
    return v;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) t[i] = e + i < C ? row[e + i] : (T)fill;
  gmk_u32x4 v;
  __builtin_memcpy(&v, t, 16);
  return v;
}

// the value at position j of an array of one of the three types, chosen at run time (the teacher's few kept logits)
__device__ __forceinline__ float gmk_load_as(const void* p, int type, int64_t j) {
  if (type == GMK_BF16) return (float)((const __bf16*)p)[j];
  if (type == GMK_F16) return (float)((const _Float16*)p)[j];
  return ((const float*)p)[j];
}

__device__ __forceinline__ float gmk_wave_max_all(float v) {   // NaN-free maximum, the result in every lane
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
// Maximum that is NaN where any value is.
__device__ __forceinline__ float gmk_wave_maximum_all(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = __builtin_elementwise_maximum(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float gmk_wave_sum_all(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Workgroup reductions over NT threads, the result in every thread; `red`: NT / 64 floats of LDS (twice that for the pair of
// sums).  A barrier on entry, so that `red` may be used by the next call at once.
template <int NT>
__device__ __forceinline__ float gmk_block_max_all(float v, float* red) {
  v = gmk_wave_max_all(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = fmaxf(r, red[i]);
  return r;
}
template <int NT>
__device__ __forceinline__ float gmk_block_maximum_all(float v, float* red) {
  v = gmk_wave_maximum_all(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = __builtin_elementwise_maximum(r, red[i]);
  return r;
}
template <int NT>
__device__ __forceinline__ void gmk_block_sum2_all(float& a, float& b, float* red) {
  a = gmk_wave_sum_all(a);
  b = gmk_wave_sum_all(b);
  if constexpr (NT == 64) return;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = a;
    red[NT / 64 + (threadIdx.x >> 6)] = b;
  }
  __syncthreads();
  a = red[0];
  b = red[NT / 64];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) {
    a += red[i];
    b += red[NT / 64 + i];
  }
}
