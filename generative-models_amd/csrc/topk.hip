// topk.hip -- the k largest of each row with their indices (the teacher's logits that are kept for distillation).  No
// counterpart in the reference.
//
// A value becomes a 32-bit key whose unsigned order is the order wanted (-0 as 0, NaN above all); with the complement of its
// index below it, a 64-bit key without ties.
#include "rows.h"
#include "quantize.h"
#include "plan.h"

typedef unsigned long long u64;

__device__ __forceinline__ unsigned topk_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);   // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One workgroup per row: the k-th largest key by four passes over the row, 8 bits of the key each (a histogram of the elements
// that agree with the bits found so far), then the elements above it, and those equal to it by rising index until k are there.
template <class T, int NT>
__device__ void topk_radix_row(const T* __restrict__ x, int64_t C, int k, T* __restrict__ value, int* __restrict__ index) {
  __shared__ unsigned hist[256];
  __shared__ u64 cand[GMK_TOPK_MAX];
  __shared__ unsigned s_bin, s_need, s_n, s_wave[NT / 64];
  const int tid = threadIdx.x;
  unsigned prefix = 0, need = (unsigned)k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    for (int64_t c = tid; c < C; c += NT) {
      const unsigned key = topk_key((float)x[c]);
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned have = 0, b = 255;
      while (have + hist[b] < need) have += hist[b--];   // the bins below hold the rest: the sum over all of them is >= need
      s_bin = b;
      s_need = need - have;
    }
    __syncthreads();
    prefix = (prefix << 8) | s_bin;
    need = s_need;
    __syncthreads();
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  // above the k-th key: k - need elements, in any order
  for (int64_t c = tid; c < C; c += NT) {
    const unsigned key = topk_key((float)x[c]);
    if (key > prefix) cand[atomicAdd(&s_n, 1u)] = ((u64)key << 32) | (0xFFFFFFFFu - (unsigned)c);
  }
  // equal to it: the first `need` by index
  unsigned base = 0;
  for (int64_t c0 = 0; c0 < C && base < need; c0 += NT) {
    const int64_t c = c0 + tid;
    const bool hit = c < C && topk_key((float)x[c]) == prefix;
    const u64 ballot = __ballot(hit);
    __syncthreads();
    if ((tid & 63) == 0) s_wave[tid >> 6] = (unsigned)__popcll(ballot);
    __syncthreads();
    unsigned before = base, all = 0;
    for (int w = 0; w < NT / 64; ++w) {
      if (w < (tid >> 6)) before += s_wave[w];
      all += s_wave[w];
    }
    before += (unsigned)__popcll(ballot & ((1ull << (tid & 63)) - 1));
    if (hit && before < need) cand[(unsigned)k - need + before] = ((u64)prefix << 32) | (0xFFFFFFFFu - (unsigned)c);
    base += all;
  }
  __syncthreads();
  // k different keys: an element's place is the number of larger ones
  for (int i = tid; i < k; i += NT) {
    const u64 mine = cand[i];
    int place = 0;
    for (int j = 0; j < k; ++j) place += cand[j] > mine;
    const unsigned c = 0xFFFFFFFFu - (unsigned)mine;
    value[place] = x[c];
    index[place] = (int)c;
  }
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void topk_rows_kernel(const T* __restrict__ x, T* __restrict__ value, int* __restrict__ index,
                                                       int64_t C, int k) {
  const int64_t row = blockIdx.x;
  topk_radix_row<T, NT>(x + row * C, C, k, value + row * k, index + row * k);
}

extern "C" size_t gmk_topk_rows_workspace_bytes(int64_t n, int64_t C, int k) { return 0; }

extern "C" int gmk_topk_rows(const void* x, int xtype, void* value, int* index, int64_t n, int64_t C, int k, void* ws,
                             size_t ws_bytes, gmk_stream_t stream) {
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(n >= 0 && n <= GMK_MAX_ROWS && C > 0 && k > 0 && k <= C, GMK_E_SHAPE);
  GMK_REQUIRE(k <= GMK_TOPK_MAX && C < 0x7FFFFFFFll, GMK_E_TOO_LARGE);
  if (n == 0) return GMK_OK;
  GMK_REQUIRE(x && value && index, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned_to(value, gmk_dtype_size(xtype)) &&
              gmk_aligned_to(index, 4), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_topk_rows_workspace_bytes(n, C, k), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_topk_rows, x, xtype, value, index, n, C, k, ws, ws_bytes, stream);
  gmk_with_dtype(xtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((topk_rows_kernel<T, 256>), dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, (const T*)x, (T*)value,
                       index, C, k);
    return 0;
  });
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}
