// distill.hip -- the loss of a student against a teacher's kept logits and against labels, with its gradient.  No counterpart in
// the reference (its classifier learns from labels alone, models/classifiers.py:86-95).
//
//   d_c = z_c - max z,  S_T = sum_c exp(d_c / T),  S_1 = sum_c exp(d_c),  p = softmax(t / T) over the row's entries
//   loss = soft T^2 (sum_j p_j (ln p_j - d_{idx_j} / T) + ln S_T) + hard (ln S_1 - d_label)
//   dz_c = soft T (exp(d_c / T) / S_T - sum_{j: idx_j = c} p_j) + hard (exp(d_c) / S_1 - [c = label])
//
// The maximum is subtracted before anything is scaled: rows of the type's lowest value give 0 and not inf - inf.
//
// A row that the registers of a workgroup hold is read once: maximum, sums and gradient from there (distill_row_kernel).  Longer rows, and
// many long ones for the loss alone, are taken in parts: the parts' maxima and sums (distill_part_kernel), then everything else, each part's workgroup joining them
// again (distill_grad_kernel, which is the backward pass too).  The gradient of the listed classes is written over what the dense pass
// wrote, by the workgroup that wrote it.
//
// Measured: 4096x32768 bf16 with labels 125 to 128 us, 4.2 TB/s in and out; without them, one exponential less for each logit and for each
// gradient, 106 us and 5.1 TB/s (a copy 5.1 to 5.5): bound by the vector units, then by memory.  1001x10007 fp32 19 us, as loss and
// backward pass 12 + 18.  256x10 5.1 us, a launch and the
// latency of its chain of loads and reductions; 9x200003 fp16 11.1 us, two launches.
#include "rows.h"
#include "plan.h"

struct DistillArgs {
  const void* t;
  const int* idx;
  const int64_t* labels;
  int64_t C;
  int k, ttype;
  float T, soft, hard;
  float at, a1;       // log2(e) / T and log2(e)
  bool need_t, need_1, same;   // S_T, S_1 are needed; S_1 is S_T (T = 1)
};

// A row's entries in LDS: class (-1: none), probability, logit less the maximum (the logit itself until that is known).
struct DistillEntries {
  __attribute__((aligned(16))) float p[GMK_DISTILL_MAX_K], z[GMK_DISTILL_MAX_K];
  __attribute__((aligned(16))) int c[GMK_DISTILL_MAX_K];   // -1 from k up to a multiple of 4
  float label_z;
  int64_t label;   // -1: none
};

struct DistillStats { float mx, st, s1; };

__device__ __forceinline__ float distill_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float distill_ln(float x) { return logf(x); }

// The first wave reads the row's entries and its label; the result, in that wave: whether any entry has weight.
template <class T>
__device__ __forceinline__ bool distill_entries(const DistillArgs& a, const T* zr, int64_t row, DistillEntries& en) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) {
    int64_t l = a.labels && a.hard != 0.f ? a.labels[row] : -1;
    if (l < 0 || l >= a.C) l = -1;
    en.label = l;
    en.label_z = l >= 0 ? (float)zr[l] : 0.f;
  }
  float mx = -__builtin_inff();
  for (int j = lane; j < ((a.k + 3) & ~3); j += 64) {
    const int c = j < a.k ? a.idx[row * a.k + j] : -1;
    const bool there = c >= 0 && c < a.C;
    const float t = there ? gmk_load_as(a.t, a.ttype, row * a.k + j) : -__builtin_inff();
    en.c[j] = there ? c : -1;
    en.z[j] = there ? (float)zr[c] : 0.f;
    en.p[j] = t;
    mx = __builtin_elementwise_maximum(mx, t);
  }
  mx = gmk_wave_maximum_all(mx);
  const bool has = mx != -__builtin_inff() && a.soft != 0.f;
  float sum = 0.f;
  for (int j = lane; j < a.k; j += 64) {
    const float e = has && en.c[j] >= 0 ? distill_exp2((en.p[j] - mx) * a.at) : 0.f;
    en.p[j] = e;
    sum += e;
  }
  sum = gmk_wave_sum_all(sum);
  const float inv = has ? 1.0f / sum : 0.f;
  for (int j = lane; j < a.k; j += 64) en.p[j] *= inv;
  return has;
}

// The row's loss, in the first wave's lanes.
__device__ __forceinline__ float distill_loss(const DistillArgs& a, const DistillEntries& en, bool has, const DistillStats& s) {
  float loss = 0.f;
  if (has) {
    float sum = 0.f;
    for (int j = threadIdx.x & 63; j < a.k; j += 64) {
      const float p = en.p[j];
      if (p != 0.f) sum += p * (distill_ln(p) - (en.z[j] - s.mx) / a.T);
    }
    loss = a.soft * a.T * a.T * (gmk_wave_sum_all(sum) + distill_ln(s.st));
  }
  if (en.label >= 0) loss += a.hard * (distill_ln(s.s1) - (en.label_z - s.mx));
  return loss;
}

// What a row's gradient is made of: dz = gt exp(d / T) + g1 exp(d) - ct p - c1 [label]
struct DistillGrad {
  float mx, gt, g1, ct, c1;
  __device__ __forceinline__ DistillGrad(const DistillArgs& a, const DistillEntries& en, bool has, const DistillStats& s, float g) {
    const bool empty = s.mx == -__builtin_inff();
    mx = empty ? 0.f : s.mx;   // then every exponential is 0
    ct = has && !empty ? g * a.soft * a.T : 0.f;
    c1 = en.label >= 0 && !empty ? g * a.hard : 0.f;
    gt = ct != 0.f ? ct / s.st : 0.f;
    g1 = c1 != 0.f ? c1 / s.s1 : 0.f;
  }
  // VEC values of a piece
  template <class T>
  __device__ __forceinline__ void piece(const DistillArgs& a, const gmk_u32x4& v, float* o) const {
    constexpr int VEC = gmk_elem<T>::VEC;
    if (gt == 0.f && g1 == 0.f) {   // a row with neither part gives zeros, whatever its logits are: NaN * 0 is none
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = 0.f;
      return;
    }
    float d[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) d[i] = gmk_piece<T>(v, i) - mx;
    if (a.same) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = distill_exp2(d[i] * a.at) * (gt + g1);
    } else if (a.need_t && a.need_1) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = fmaf(distill_exp2(d[i] * a.a1), g1, distill_exp2(d[i] * a.at) * gt);
    } else if (a.need_t) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = distill_exp2(d[i] * a.at) * gt;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = distill_exp2(d[i] * a.a1) * g1;
    }
  }
};

// The first wave writes the gradient of the listed classes in [from, to) and of the label, whole: entries of the same class write the
// same value.  dzr: the row's gradient at class 0.
template <class T>
__device__ __forceinline__ void distill_listed(const DistillArgs& a, const DistillEntries& en, const DistillGrad& g, T* dzr, int64_t from, int64_t to) {
  for (int j = threadIdx.x & 63; j <= a.k; j += 64) {
    const bool is_label = j == a.k;
    const int64_t c = is_label ? (g.c1 != 0.f ? en.label : -1) : (g.ct != 0.f ? en.c[j] : -1);
    if (c < from || c >= to) continue;
    float p = 0.f;
    if (g.ct != 0.f)
#pragma unroll 4
      for (int i = 0; i < a.k; i += 4) {
        const int4 ci = *(const int4*)(en.c + i);
        const float4 pi = *(const float4*)(en.p + i);
        p += (ci.x == c ? pi.x : 0.f) + (ci.y == c ? pi.y : 0.f) + (ci.z == c ? pi.z : 0.f) + (ci.w == c ? pi.w : 0.f);
      }
    const float d = (is_label ? en.label_z : en.z[j]) - g.mx;
    float r = g.gt != 0.f ? fmaf(distill_exp2(d * a.at), g.gt, -g.ct * p) : 0.f;
    if (g.g1 != 0.f) r += fmaf(distill_exp2(d * a.a1), g.g1, c == en.label ? -g.c1 : 0.f);
    dzr[c] = (T)r;
  }
}

// sums of exponentials of a piece, into two chains each
template <class T>
__device__ __forceinline__ void distill_sums(const DistillArgs& a, const gmk_u32x4& v, float mx, float* st, float* s1) {
  constexpr int VEC = gmk_elem<T>::VEC;
  float d[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) d[i] = gmk_piece<T>(v, i) - mx;
  if (a.need_t) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) st[i & 1] += distill_exp2(d[i] * a.at);
  }
  if (a.need_1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) s1[i & 1] += distill_exp2(d[i] * a.a1);
  }
}
template <class T>
__device__ __forceinline__ float distill_most(const gmk_u32x4& v, float mx) {
#pragma unroll
  for (int i = 0; i < gmk_elem<T>::VEC; ++i) mx = __builtin_elementwise_maximum(mx, gmk_piece<T>(v, i));
  return mx;
}

// Elements [e, C) of a row from a piece's values, as far as there are any.  `stream`: whole pieces go past the caches, where the logits stay.
// For the backward pass and rows in parts always (with the loss before it 4096x32768 bf16 188 us, else 201; 8000x8001 fp16 93.2, else 99.8;
// 400x200003 fp16 in parts 101, else 113.5); for a row in registers, where the logits have no more use, if rows are whole lines of 128 bytes
// (4096x32768 bf16 128, else 135; 8000x8001 fp16 would take 67, else 62).
template <class T>
__device__ __forceinline__ void distill_put(T* dzr, int64_t e, int64_t C, const float* o, bool stream) {
  constexpr int VEC = gmk_elem<T>::VEC;
  if (e + VEC <= C) {
    if (stream) gmk_store16<true>(dzr + e, gmk_pack<T>(o));
    else gmk_store16<false>(dzr + e, gmk_pack<T>(o));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (e + i < C) dzr[e + i] = (T)o[i];
  }
}

// Loss (MODE 0: and stats; MODE 2: and gradient) of a row that NT * KEEP pieces of 16 bytes hold.
template <class T, int NT, int KEEP, int MODE>
__global__ __launch_bounds__(NT) void distill_row_kernel(const T* __restrict__ z, DistillArgs a, const float* __restrict__ weight, float scale,
                                                         float* __restrict__ loss, float* __restrict__ stats, T* __restrict__ dz) {
  constexpr int VEC = gmk_elem<T>::VEC;
  __shared__ float red[2 * NT / 64];
  __shared__ DistillEntries en;
  __shared__ int s_has;
  const int64_t row = blockIdx.x;
  const T* zr = z + row * a.C;
  T* dzr = dz + row * a.C;
  const int64_t e0 = (int64_t)threadIdx.x * VEC;
  const bool lines = (((uintptr_t)dz | (uintptr_t)(a.C * (int64_t)sizeof(T))) & 127) == 0;
  const float w = MODE == 2 && weight ? weight[row] : 1.f;
  if (MODE == 2 && w == 0.f) {
    float o[VEC] = {};
#pragma unroll
    for (int i = 0; i < KEEP; ++i) distill_put(dzr, e0 + (int64_t)i * NT * VEC, a.C, o, lines);
    if (threadIdx.x == 0) loss[row] = 0.f;
    return;
  }
  gmk_u32x4 keep[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) keep[i] = gmk_row_piece(zr, e0 + (int64_t)i * NT * VEC, a.C);
  if (threadIdx.x < 64) {
    const bool has = distill_entries(a, zr, row, en);
    if (threadIdx.x == 0) s_has = has;
  }
  if (NT == 64) __syncthreads();   // the reductions of a single wave have no barrier
  DistillStats s = {-__builtin_inff(), 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < KEEP; ++i) s.mx = distill_most<T>(keep[i], s.mx);
  s.mx = gmk_block_maximum_all<NT>(s.mx, red);
  if (s.mx != -__builtin_inff()) {
    float st[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KEEP; ++i) distill_sums<T>(a, keep[i], s.mx, st, s1);
    s.st = st[0] + st[1];
    s.s1 = s1[0] + s1[1];
  }
  gmk_block_sum2_all<NT>(s.st, s.s1, red);
  if (a.same) s.s1 = s.st;
  const bool has = s_has;
  if (threadIdx.x < 64) {
    const float l = s.mx == -__builtin_inff() ? 0.f : distill_loss(a, en, has, s);
    if (threadIdx.x == 0) {
      loss[row] = w * l;
      if (MODE == 0) {
        stats[row * 3] = s.mx;
        stats[row * 3 + 1] = s.st;
        stats[row * 3 + 2] = s.s1;
      }
    }
  }
  if constexpr (MODE == 2) {
    const DistillGrad g(a, en, has, s, w * scale);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      float o[VEC];
      g.piece<T>(a, keep[i], o);
      distill_put(dzr, e0 + (int64_t)i * NT * VEC, a.C, o, lines);
    }
    __syncthreads();
    if (threadIdx.x < 64) distill_listed(a, en, g, dzr, 0, a.C);
  }
}

#define DISTILL_NT 256
#define DISTILL_KEEP 4   // pieces of a part's thread

// part blockIdx.x % parts of row blockIdx.x / parts -> its maximum and sums
template <class T>
__global__ __launch_bounds__(DISTILL_NT) void distill_part_kernel(const T* __restrict__ z, DistillArgs a, const float* __restrict__ weight,
                                                                  float* __restrict__ part, unsigned parts) {
  constexpr int VEC = gmk_elem<T>::VEC, NT = DISTILL_NT, KEEP = DISTILL_KEEP;
  __shared__ float red[2 * NT / 64];
  const int64_t row = blockIdx.x / parts, from = (int64_t)(blockIdx.x % parts) * NT * KEEP * VEC;
  if (weight && weight[row] == 0.f) return;
  const T* zr = z + row * a.C;
  const int64_t e0 = from + (int64_t)threadIdx.x * VEC;
  gmk_u32x4 keep[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) keep[i] = gmk_row_piece(zr, e0 + i * NT * VEC, a.C);
  DistillStats s = {-__builtin_inff(), 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < KEEP; ++i) s.mx = distill_most<T>(keep[i], s.mx);
  s.mx = gmk_block_maximum_all<NT>(s.mx, red);
  if (s.mx != -__builtin_inff()) {
    float st[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KEEP; ++i) distill_sums<T>(a, keep[i], s.mx, st, s1);
    s.st = st[0] + st[1];
    s.s1 = s1[0] + s1[1];
  }
  gmk_block_sum2_all<NT>(s.st, s.s1, red);
  if (threadIdx.x == 0) {
    float* p = part + (int64_t)blockIdx.x * 3;
    p[0] = s.mx;
    p[1] = s.st;
    p[2] = s.s1;
  }
}

// a row's maximum and sums from its parts', in every thread (a fixed order: every workgroup of the row gets the same); `mine`: those of part
// threadIdx.x, loaded before
template <int NT>
__device__ __forceinline__ DistillStats distill_join(const DistillArgs& a, const DistillStats& mine, const float* __restrict__ part, unsigned parts, float* red) {
  DistillStats s = {mine.mx, 0.f, 0.f};
  for (unsigned i = threadIdx.x + NT; i < parts; i += NT) s.mx = __builtin_elementwise_maximum(s.mx, part[3 * (int64_t)i]);
  s.mx = gmk_block_maximum_all<NT>(s.mx, red);
  if (s.mx != -__builtin_inff()) {
    s.st = mine.st * distill_exp2((mine.mx - s.mx) * a.at);
    s.s1 = mine.s1 * distill_exp2((mine.mx - s.mx) * a.a1);
    for (unsigned i = threadIdx.x + NT; i < parts; i += NT) {
      const float d = part[3 * (int64_t)i] - s.mx;
      s.st += part[3 * (int64_t)i + 1] * distill_exp2(d * a.at);
      s.s1 += part[3 * (int64_t)i + 2] * distill_exp2(d * a.a1);
    }
  }
  gmk_block_sum2_all<NT>(s.st, s.s1, red);
  if (a.same) s.s1 = s.st;
  return s;
}

// MODE 0: loss and stats of a row from its parts; MODE 1: gradient of a part from stats; MODE 2: gradient of a part, and the loss with the
// first one, from the row's parts.  `from_parts`: the row's parts (0, 2) or its stats (1).
template <class T, int NT, int MODE>
__global__ __launch_bounds__(NT) void distill_grad_kernel(const T* __restrict__ z, DistillArgs a, const float* __restrict__ weight, float scale,
                                                          const float* __restrict__ from_parts, unsigned parts, float* __restrict__ loss,
                                                          float* __restrict__ stats, T* __restrict__ dz) {
  constexpr int VEC = gmk_elem<T>::VEC, KEEP = DISTILL_KEEP;
  __shared__ float red[2 * NT / 64];
  __shared__ DistillEntries en;
  __shared__ int s_has;
  const unsigned blocks = MODE == 0 ? 1 : parts;   // workgroups of a row
  const int64_t row = blockIdx.x / blocks, from = (int64_t)(blockIdx.x % blocks) * NT * KEEP * VEC;
  const T* zr = z + row * a.C;
  T* dzr = dz + row * a.C;
  const int64_t e0 = from + (int64_t)threadIdx.x * VEC;
  const float w = MODE != 0 && weight ? weight[row] : 1.f;
  if (MODE != 0 && w == 0.f) {
    float o[VEC] = {};
#pragma unroll
    for (int i = 0; i < KEEP; ++i) distill_put(dzr, e0 + i * NT * VEC, a.C, o, true);
    if (MODE == 2 && from == 0 && threadIdx.x == 0) loss[row] = 0.f;
    return;
  }
  gmk_u32x4 keep[KEEP];
  if constexpr (MODE != 0) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) keep[i] = gmk_row_piece(zr, e0 + i * NT * VEC, a.C);
  }
  DistillStats s = {-__builtin_inff(), 0.f, 0.f};
  if (MODE != 1 && threadIdx.x < parts) {
    const float* p = from_parts + (row * parts + threadIdx.x) * 3;
    s = {p[0], p[1], p[2]};
  }
  if (threadIdx.x < 64) {
    const bool has = distill_entries(a, zr, row, en);
    if (threadIdx.x == 0) s_has = has;
  }
  if constexpr (MODE == 1) {
    s = {from_parts[row * 3], from_parts[row * 3 + 1], from_parts[row * 3 + 2]};
    __syncthreads();
  } else {
    s = distill_join<NT>(a, s, from_parts + row * parts * 3, parts, red);
    if (NT == 64) __syncthreads();
  }
  const bool has = s_has;
  if (MODE != 1 && from == 0 && threadIdx.x < 64) {
    const float l = s.mx == -__builtin_inff() ? 0.f : distill_loss(a, en, has, s);
    if (threadIdx.x == 0) {
      loss[row] = w * l;
      if (MODE == 0) {
        stats[row * 3] = s.mx;
        stats[row * 3 + 1] = s.st;
        stats[row * 3 + 2] = s.s1;
      }
    }
  }
  if constexpr (MODE != 0) {
    const DistillGrad g(a, en, has, s, w * scale);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      float o[VEC];
      g.piece<T>(a, keep[i], o);
      distill_put(dzr, e0 + i * NT * VEC, a.C, o, true);
    }
    __syncthreads();
    if (threadIdx.x < 64) distill_listed(a, en, g, dzr, from, from + (int64_t)NT * KEEP * VEC);
  }
}

static int64_t distill_parts(int64_t C, int vec) { return (C + DISTILL_NT * DISTILL_KEEP * vec - 1) / (DISTILL_NT * DISTILL_KEEP * vec); }

// Rows in parts: those that no workgroup's registers hold (8 pieces for each of 1024 threads), and, for the loss alone, many that only a
// workgroup of 1024 threads would: 2048x65536 bf16 55 us in parts, whole rows 94; 512x49000 17.7 (20.1; the same with 511 rows, which are
// taken whole).  With the gradient whole rows win, as they are read once: 512x49000 37.2 us, in parts it would take 40.6.
static bool distill_in_parts(int mode, int64_t n, int64_t C, int vec) {
  const int64_t pieces = (C + vec - 1) / vec;
  return pieces > 8192 || (mode == 0 && n >= 512 && pieces > 4096);
}

extern "C" size_t gmk_distill_workspace_bytes(int64_t n, int64_t C) {
  if (n <= 0 || C <= 0) return 0;
  return distill_in_parts(0, n, C, 4) || distill_in_parts(0, n, C, 8) ? (size_t)n * distill_parts(C, 4) * 12 : 0;
}

static int distill_check(int ztype, int ttype, int64_t n, int64_t C, int k, float T, float soft, float hard) {
  GMK_REQUIRE(gmk_dtype_ok(ztype) && gmk_dtype_ok(ttype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(T >= GMK_DISTILL_MIN_T && T <= GMK_DISTILL_MAX_T && soft - soft == 0.f && hard - hard == 0.f, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(n >= 0 && C > 0 && k > 0, GMK_E_SHAPE);
  GMK_REQUIRE(k <= GMK_DISTILL_MAX_K && C < 0x7FFFFFFFll, GMK_E_TOO_LARGE);
  return GMK_OK;
}

static DistillArgs distill_args(const void* t, int ttype, const int* idx, const int64_t* labels, int64_t C, int k, float T, float soft, float hard) {
  const float log2e = 1.44269504088896340736f;
  DistillArgs a{t, idx, labels, C, k, ttype, T, soft, hard, log2e / T, log2e, soft != 0.f, labels && hard != 0.f, false};
  a.same = a.need_t && a.need_1 && T == 1.f;
  if (a.same) a.need_1 = false;
  return a;
}

// MODE 0: loss and stats; 2: loss and gradient
template <int MODE>
static int distill_launch(const void* z, int ztype, const DistillArgs& a, const float* weight, float scale, float* loss, float* stats, void* dz,
                          int64_t n, void* ws, hipStream_t stream) {
  return gmk_with_dtype(ztype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int VEC = gmk_elem<T>::VEC;
    if (distill_in_parts(MODE, n, a.C, VEC)) {
      const int64_t parts = distill_parts(a.C, VEC);
      GMK_REQUIRE(gmk_grid_ok(n * parts, DISTILL_NT), GMK_E_TOO_LARGE);
      hipLaunchKernelGGL((distill_part_kernel<T>), dim3((unsigned)(n * parts)), dim3(DISTILL_NT), 0, stream, (const T*)z, a, weight, (float*)ws, (unsigned)parts);
      GMK_CHECK_LAUNCH();
      constexpr int NT = MODE == 0 ? 64 : DISTILL_NT;   // the loss alone is a wave's work
      hipLaunchKernelGGL((distill_grad_kernel<T, NT, MODE>), dim3((unsigned)(MODE == 0 ? n : n * parts)), dim3(NT), 0, stream, (const T*)z, a, weight, scale,
                         (const float*)ws, (unsigned)parts, loss, stats, (T*)dz);
      GMK_CHECK_LAUNCH();
      return GMK_OK;
    }
    auto go = [&](auto kernel, int threads) -> int {
      GMK_REQUIRE(gmk_grid_ok(n, threads), GMK_E_TOO_LARGE);
      hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), 0, stream, (const T*)z, a, weight, scale, loss, stats, (T*)dz);
      GMK_CHECK_LAUNCH();
      return GMK_OK;
    };
    const int64_t pieces = (a.C + VEC - 1) / VEC;
    // As few pieces a thread as hold the row (one that no thread has costs what the others do: 4096x20000 bf16 with labels 81 us with 10 of
    // 256 threads, 118 with 6 of 512 and 129 with 8; 2048x36000 136 with 6 of 1024, 155 with 8), and as few threads, so that several workgroups of a
    // unit are at different steps (5 of 512 threads would take 86; without labels 71, 10 of 256 75.5).
    if (pieces <= 64 * 1) return go(distill_row_kernel<T, 64, 1, MODE>, 64);
    if (pieces <= 64 * 2) return go(distill_row_kernel<T, 64, 2, MODE>, 64);
    if (pieces <= 64 * 4) return go(distill_row_kernel<T, 64, 4, MODE>, 64);
    if (pieces <= 256 * 2) return go(distill_row_kernel<T, 256, 2, MODE>, 256);
    if (pieces <= 256 * 4) return go(distill_row_kernel<T, 256, 4, MODE>, 256);
    if (pieces <= 256 * 6) return go(distill_row_kernel<T, 256, 6, MODE>, 256);
    if (pieces <= 256 * 8) return go(distill_row_kernel<T, 256, 8, MODE>, 256);
    if (pieces <= 256 * 10) return go(distill_row_kernel<T, 256, 10, MODE>, 256);
    if (pieces <= 512 * 6) return go(distill_row_kernel<T, 512, 6, MODE>, 512);
    if (pieces <= 512 * 7) return go(distill_row_kernel<T, 512, 7, MODE>, 512);
    if (pieces <= 512 * 8) return go(distill_row_kernel<T, 512, 8, MODE>, 512);
    if (pieces <= 1024 * 6) return go(distill_row_kernel<T, 1024, 6, MODE>, 1024);
    return go(distill_row_kernel<T, 1024, 8, MODE>, 1024);
  });
}

// the gradient from stats
static int distill_bwd_launch(const void* z, int ztype, const DistillArgs& a, const float* grad, const float* stats, void* dz, int64_t n, hipStream_t stream) {
  return gmk_with_dtype(ztype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int VEC = gmk_elem<T>::VEC;
    const bool small = a.C <= 64 * DISTILL_KEEP * VEC;
    const int64_t parts = small ? 1 : distill_parts(a.C, VEC);
    GMK_REQUIRE(gmk_grid_ok(n * parts, DISTILL_NT), GMK_E_TOO_LARGE);
    if (small) hipLaunchKernelGGL((distill_grad_kernel<T, 64, 1>), dim3((unsigned)n), dim3(64), 0, stream, (const T*)z, a, grad, 1.f, stats, 1u, nullptr, nullptr, (T*)dz);
    else hipLaunchKernelGGL((distill_grad_kernel<T, DISTILL_NT, 1>), dim3((unsigned)(n * parts)), dim3(DISTILL_NT), 0, stream, (const T*)z, a, grad, 1.f, stats, (unsigned)parts, nullptr, nullptr, (T*)dz);
    GMK_CHECK_LAUNCH();
    return GMK_OK;
  });
}

extern "C" int gmk_distill_fwd(const void* z, int ztype, const void* t, int ttype, const int* idx, const int64_t* labels,
                               float* loss, float* stats, int64_t n, int64_t C, int k, float T, float soft, float hard, void* ws,
                               size_t ws_bytes, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(z && t && idx && loss && stats && (ws || gmk_distill_workspace_bytes(n, C) == 0), GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) &&
              gmk_aligned_to(labels, 8) && gmk_aligned_to(loss, 4) && gmk_aligned_to(stats, 4) && gmk_aligned16(ws), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_distill_workspace_bytes(n, C), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_distill_fwd, z, ztype, t, ttype, idx, labels, loss, stats, n, C, k, T, soft, hard, ws, ws_bytes, stream);
  return distill_launch<0>(z, ztype, distill_args(t, ttype, idx, labels, C, k, T, soft, hard), nullptr, 1.f, loss, stats, nullptr, n, ws, (hipStream_t)stream);
}

extern "C" int gmk_distill_bwd(const float* grad, const void* z, int ztype, const void* t, int ttype, const int* idx,
                               const int64_t* labels, const float* stats, void* dz, int64_t n, int64_t C, int k, float T,
                               float soft, float hard, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(grad && z && t && idx && stats && dz, GMK_E_NULL);
  GMK_REQUIRE(dz != z, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(dz, gmk_dtype_size(ztype)) &&
              gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) && gmk_aligned_to(labels, 8) &&
              gmk_aligned_to(grad, 4) && gmk_aligned_to(stats, 4), GMK_E_ALIGN);
  GMK_PLAN_HOOK(gmk_distill_bwd, grad, z, ztype, t, ttype, idx, labels, stats, dz, n, C, k, T, soft, hard, stream);
  return distill_bwd_launch(z, ztype, distill_args(t, ttype, idx, labels, C, k, T, soft, hard), grad, stats, dz, n, (hipStream_t)stream);
}

extern "C" int gmk_distill_fwd_bwd(const void* z, int ztype, const void* t, int ttype, const int* idx, const int64_t* labels,
                                   const float* weight, float* loss, void* dz, int64_t n, int64_t C, int k, float T, float soft,
                                   float hard, float scale, void* ws, size_t ws_bytes, gmk_stream_t stream) {
  const int rc = distill_check(ztype, ttype, n, C, k, T, soft, hard);
  if (rc != GMK_OK) return rc;
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(z && t && idx && loss && dz && (ws || gmk_distill_workspace_bytes(n, C) == 0), GMK_E_NULL);
  GMK_REQUIRE(dz != z, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(gmk_aligned_to(z, gmk_dtype_size(ztype)) && gmk_aligned_to(dz, gmk_dtype_size(ztype)) &&
              gmk_aligned_to(t, gmk_dtype_size(ttype)) && gmk_aligned_to(idx, 4) && gmk_aligned_to(labels, 8) &&
              gmk_aligned_to(weight, 4) && gmk_aligned_to(loss, 4) && gmk_aligned16(ws), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_distill_workspace_bytes(n, C), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_distill_fwd_bwd, z, ztype, t, ttype, idx, labels, weight, loss, dz, n, C, k, T, soft, hard, scale, ws, ws_bytes, stream);
  return distill_launch<2>(z, ztype, distill_args(t, ttype, idx, labels, C, k, T, soft, hard), weight, scale, loss, nullptr, dz, n, ws, (hipStream_t)stream);
}
