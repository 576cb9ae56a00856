// distill.hip -- the loss of a student against a teacher's kept logits and against labels, with its gradient.  No counterpart in
// the reference (its classifier learns from labels alone, models/classifiers.py:86-95).
//
//   d_c = z_c - max z,  S_T = sum_c exp(d_c / T),  S_1 = sum_c exp(d_c),  p = softmax(t / T) over the row's entries
//   loss = soft T^2 (sum_j p_j (ln p_j - d_{idx_j} / T) + ln S_T) + hard (ln S_1 - d_label)
//   dz_c = soft T (exp(d_c / T) / S_T - sum_{j: idx_j = c} p_j) + hard (exp(d_c) / S_1 - [c = label])
//
// The maximum is subtracted before anything is scaled: rows of the type's lowest value give 0 and not inf - inf.
#include "rows.h"
#include "quantize.h"
#include "plan.h"

struct DistillArgs {
  const void* t;
  const int* idx;
  const int64_t* labels;
  int64_t C;
  int k, ttype;
  float T, soft, hard;
};

// What a row of entries comes to, in LDS: their classes and probabilities.
struct DistillEntries {
  float p[GMK_DISTILL_MAX_K];
  int c[GMK_DISTILL_MAX_K];
};

// The first wave reads the row's entries and leaves them in `en`; the result, in that wave: whether any has weight.
__device__ __forceinline__ bool distill_entries(const DistillArgs& a, int64_t row, DistillEntries& en) {
  const int lane = threadIdx.x & 63;
  float mx = -__builtin_inff();
  bool nan = false;
  for (int j = lane; j < a.k; j += 64) {
    const int c = a.idx[row * a.k + j];
    const bool there = c >= 0 && c < a.C;
    const float t = there ? gmk_load_as(a.t, a.ttype, row * a.k + j) : -__builtin_inff();
    en.c[j] = there ? c : -1;
    en.p[j] = t;
    nan |= t != t;
    mx = fmaxf(mx, t);
  }
  mx = gmk_wave_max_all(mx);
  if (__any(nan)) mx = __builtin_nanf("");
  const bool has = mx != -__builtin_inff();
  float sum = 0.f;
  for (int j = lane; j < a.k; j += 64) {
    const float e = has && en.c[j] >= 0 ? expf((en.p[j] - mx) / a.T) : 0.f;
    en.p[j] = e;
    sum += e;
  }
  sum = gmk_wave_sum_all(sum);
  for (int j = lane; j < a.k; j += 64) en.p[j] = has ? en.p[j] / sum : 0.f;
  return has;
}

// The row's loss, in the first wave's lanes, from its maximum and its sums.
template <class T>
__device__ __forceinline__ float distill_row_loss(const DistillArgs& a, const T* zr, int64_t row, const DistillEntries& en,
                                                  bool has, float mx, float st, float s1) {
  float loss = 0.f;
  if (has && a.soft != 0.f) {
    float s = 0.f;
    for (int j = threadIdx.x & 63; j < a.k; j += 64) {
      const float p = en.p[j];
      if (p != 0.f) s += p * (logf(p) - ((float)zr[en.c[j]] - mx) / a.T);
    }
    loss = a.soft * a.T * a.T * (gmk_wave_sum_all(s) + logf(st));
  }
  if (a.labels && a.hard != 0.f) {
    const int64_t l = a.labels[row];
    if (l >= 0 && l < a.C) loss += a.hard * (logf(s1) - ((float)zr[l] - mx));
  }
  return loss;
}

// The gradient of the classes that are listed, over what the dense pass wrote: each is computed whole, and entries of the same
// class write the same value.
template <class T>
__device__ __forceinline__ void distill_listed(const DistillArgs& a, const T* zr, T* dzr, const DistillEntries& en, bool has,
                                               int64_t label, float mx, float gt, float g1, float ct, float c1) {
  for (int j = threadIdx.x & 63; j <= a.k; j += 64) {
    const int64_t c = j < a.k ? (has ? en.c[j] : -1) : label;
    if (c < 0) continue;
    float p = 0.f;
    if (has)
      for (int i = 0; i < a.k; ++i) p += en.c[i] == c ? en.p[i] : 0.f;
    const float d = (float)zr[c] - mx;
    float g = gt != 0.f ? fmaf(expf(d / a.T), gt, -ct * p) : 0.f;
    if (g1 != 0.f) g += fmaf(expf(d), g1, c == label ? -c1 : 0.f);
    dzr[c] = (T)g;
  }
}

// MODE 0: loss and stats; 1: gradient from stats; 2: both.  One workgroup per row, which passes over the row up to three times.
template <class T, int NT, int MODE>
__global__ __launch_bounds__(NT) void distill_kernel(const T* __restrict__ z, DistillArgs a, const float* __restrict__ weight,
                                                     float scale, float* __restrict__ loss, float* stats, T* __restrict__ dz) {
  constexpr int VEC = gmk_elem<T>::VEC;
  __shared__ float red[2 * NT / 64];
  __shared__ DistillEntries en;
  __shared__ int s_has;
  const int64_t row = blockIdx.x;
  const T* zr = z + row * a.C;
  const float w = MODE != 0 && weight ? weight[row] : 1.f;
  if (MODE != 0 && w == 0.f) {
    const gmk_u32x4 zero = {0u, 0u, 0u, 0u};
    for (int64_t e = (int64_t)threadIdx.x * VEC; e < a.C; e += NT * VEC) {
      if (e + VEC <= a.C) gmk_store16(dz + row * a.C + e, zero);
      else for (int64_t c = e; c < a.C; ++c) dz[row * a.C + c] = (T)0.f;
    }
    if (MODE == 2 && threadIdx.x == 0) loss[row] = 0.f;
    return;
  }
  if (threadIdx.x < 64) {
    const bool has = distill_entries(a, row, en);
    if (threadIdx.x == 0) s_has = has;
  }
  float mx, st = 0.f, s1 = 0.f;
  if (MODE == 1) {
    mx = stats[row * 3];
    st = stats[row * 3 + 1];
    s1 = stats[row * 3 + 2];
    __syncthreads();
  } else {
    mx = -__builtin_inff();
    bool nan = false;
    for (int64_t e = (int64_t)threadIdx.x * VEC; e < a.C; e += NT * VEC) {
      const gmk_u32x4 v = gmk_row_piece(zr, e, a.C);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float f = gmk_piece<T>(v, i);
        nan |= f != f;
        mx = fmaxf(mx, f);
      }
    }
    mx = gmk_block_max_all<NT>(mx, red);
    if (__syncthreads_or(nan)) mx = __builtin_nanf("");
    if (mx != -__builtin_inff()) {
      for (int64_t e = (int64_t)threadIdx.x * VEC; e < a.C; e += NT * VEC) {
        const gmk_u32x4 v = gmk_row_piece(zr, e, a.C);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = gmk_piece<T>(v, i) - mx;
          st += expf(d / a.T);
          s1 += expf(d);
        }
      }
    }
    gmk_block_sum2_all<NT>(st, s1, red);
  }
  const bool empty = mx == -__builtin_inff();
  const bool has = s_has;
  if (MODE != 1 && threadIdx.x < 64) {
    const float l = empty ? 0.f : distill_row_loss<T>(a, zr, row, en, has, mx, st, s1);
    if (threadIdx.x == 0) {
      loss[row] = w * l;
      if (MODE == 0) {
        stats[row * 3] = mx;
        stats[row * 3 + 1] = st;
        stats[row * 3 + 2] = s1;
      }
    }
  }
  if (MODE == 0) return;
  const float g = w * scale;
  int64_t label = a.labels && a.hard != 0.f ? a.labels[row] : -1;
  if (label < 0 || label >= a.C) label = -1;
  const float ct = has && !empty ? g * a.soft * a.T : 0.f, c1 = label >= 0 && !empty ? g * a.hard : 0.f;
  const float gt = ct != 0.f ? ct / st : 0.f, g1 = c1 != 0.f ? c1 / s1 : 0.f;
  T* dzr = dz + row * a.C;
  for (int64_t e = (int64_t)threadIdx.x * VEC; e < a.C; e += NT * VEC) {
    const gmk_u32x4 v = gmk_row_piece(zr, e, a.C);
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = gmk_piece<T>(v, i) - mx;
      float r = 0.f;
      if (gt != 0.f) r = expf(d / a.T) * gt;
      if (g1 != 0.f) r = fmaf(expf(d), g1, r);
      o[i] = r;
    }
    const gmk_u32x4 u = gmk_pack<T>(o);
    if (e + VEC <= a.C) {
      gmk_store16(dzr + e, u);
    } else {
      for (int i = 0; e + i < a.C; ++i) dzr[e + i] = (T)o[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) distill_listed<T>(a, zr, dzr, en, has && !empty, empty ? -1 : label, mx, gt, g1, ct, c1);
}

extern "C" size_t gmk_distill_workspace_bytes(int64_t n, int64_t C) { return 0; }

static int distill_check(int ztype, int ttype, int64_t n, int64_t C, int k, float T, float soft, float hard) {
  GMK_REQUIRE(gmk_dtype_ok(ztype) && gmk_dtype_ok(ttype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(T > 0.f && T < __builtin_inff() && soft - soft == 0.f && hard - hard == 0.f, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(n >= 0 && n <= GMK_MAX_ROWS && C > 0 && k > 0, GMK_E_SHAPE);
  GMK_REQUIRE(k <= GMK_DISTILL_MAX_K && C < 0x7FFFFFFFll, GMK_E_TOO_LARGE);
  return GMK_OK;
}

template <int MODE>
static int distill_launch(const void* z, int ztype, const DistillArgs& a, const float* weight, float scale, float* loss,
                          float* stats, void* dz, int64_t n, gmk_stream_t stream) {
  gmk_with_dtype(ztype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((distill_kernel<T, 256, MODE>), dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, (const T*)z, a,
                       weight, scale, loss, stats, (T*)dz);
    return 0;
  });
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}

extern "C" int gmk_distill_fwd(const void* z, int ztype, const void* t, int ttype, const int* idx, const int64_t* labels,
                               float* loss, float* stats, int64_t n, int64_t C, int k, float T, float soft, float hard, void* ws,
                               size_t ws_bytes, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(z && t && idx && loss && stats, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) &&
              gmk_aligned_to(labels, 8) && gmk_aligned_to(loss, 4) && gmk_aligned_to(stats, 4), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_distill_workspace_bytes(n, C), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_distill_fwd, z, ztype, t, ttype, idx, labels, loss, stats, n, C, k, T, soft, hard, ws, ws_bytes, stream);
  return distill_launch<0>(z, ztype, DistillArgs{t, idx, labels, C, k, ttype, T, soft, hard}, nullptr, 1.f, loss, stats, nullptr, n, stream);
}

extern "C" int gmk_distill_bwd(const float* grad, const void* z, int ztype, const void* t, int ttype, const int* idx,
                               const int64_t* labels, const float* stats, void* dz, int64_t n, int64_t C, int k, float T,
                               float soft, float hard, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(grad && z && t && idx && stats && dz, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(dz, gmk_dtype_size(ztype)) &&
              gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) && gmk_aligned_to(labels, 8) &&
              gmk_aligned_to(grad, 4) && gmk_aligned_to(stats, 4), GMK_E_ALIGN);
  GMK_PLAN_HOOK(gmk_distill_bwd, grad, z, ztype, t, ttype, idx, labels, stats, dz, n, C, k, T, soft, hard, stream);
  return distill_launch<1>(z, ztype, DistillArgs{t, idx, labels, C, k, ttype, T, soft, hard}, grad, 1.f, nullptr, const_cast<float*>(stats), dz, n, stream);
}

extern "C" int gmk_distill_fwd_bwd(const void* z, int ztype, const void* t, int ttype, const int* idx, const int64_t* labels,
                                   const float* weight, float* loss, void* dz, int64_t n, int64_t C, int k, float T, float soft,
                                   float hard, float scale, void* ws, size_t ws_bytes, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(z && t && idx && loss && dz, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(dz, gmk_dtype_size(ztype)) &&
              gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) && gmk_aligned_to(labels, 8) &&
              gmk_aligned_to(weight, 4) && gmk_aligned_to(loss, 4), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_distill_workspace_bytes(n, C), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_distill_fwd_bwd, z, ztype, t, ttype, idx, labels, weight, loss, dz, n, C, k, T, soft, hard, scale, ws, ws_bytes, stream);
  return distill_launch<2>(z, ztype, DistillArgs{t, idx, labels, C, k, ttype, T, soft, hard}, weight, scale, loss, nullptr, dz, n, stream);
}
