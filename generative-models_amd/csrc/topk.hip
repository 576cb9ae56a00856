// topk.hip -- the k largest of each row with their indices (the teacher's logits that are kept for distillation).  No
// counterpart in the reference.
//
// A value becomes a 32-bit key whose unsigned order is the order wanted (-0 as 0, NaN above all); with the complement of its
// index below it, a 64-bit key without ties.
//
// A row is read once.  Every thread goes through its elements in segments and keeps each segment's largest; the k-th largest of the
// threads' maxima is a lower bound of the row's k-th largest element, and a close one, as the maxima are at least twice k.  Only the
// segments that reach it are read again, their elements that do are collected (k and a few more, in any order), and each finds its place
// by counting the larger ones.  Where they do not fit (many equal values at the border, or rows made to defeat this) the k-th largest
// key is found by its bits instead, 8 at a time: topk_radix_row.
// Few long rows are split into parts, one workgroup each, whose sorted lists a second launch merges.
//
// Measured: 2048x65536 bf16, k = 32 54.4 us, 4.9 TB/s of the rows' bytes, which is what a maximum over them reads at; 256x1000 fp32, k = 10
// 4.7 us and 5x150001 fp32, k = 50 11.6 us, the latency of one and of two launches' chains of loads, search and counting.  What
// is read again grows with k: 512x200000 fp16 40.4 us with k = 10 (5.1 TB/s), 59.7 with k = 128.
//
// What defeats it: a row or part whose k-th largest thread's maximum is a value that most of its elements have, as the mask's where fewer than
// k threads hold a class that is not masked.  Every element is then collected, they do not fit, and the search by bits takes five passes in
// which they all count in one bin.  5x150001 fp32, k = 50: 11.5 us, with the last tenth masked, which fills whole parts, 53, with all but the
// first 40 classes masked 73 (-inf) or 103 (the lowest value), with equal values 91.  In whole rows a masked tenth or half costs nothing, but
// with all but the first 40 classes masked, which few threads hold, 2048x65536 bf16, k = 32 takes 1184 us for 54.5, with equal values 1978;
// 300x60000 fp32, k = 50 499 and 522 for 17.6.  Up to 1024 elements do fit: 256x1000 fp32, k = 10 with equal values 41.5 for 4.7.
#include "rows.h"
#include "plan.h"

typedef unsigned long long u64;

__device__ __forceinline__ unsigned topk_key(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);   // -0 + 0 = +0
  const unsigned key = b ^ (unsigned)((int)b >> 31 | 0x80000000);
  return v != v ? 0xFFFFFFFFu : key;
}
__device__ __forceinline__ float topk_value(unsigned key) {   // of a key; a NaN for those above +inf's
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 topk_pair(unsigned key, unsigned c) { return (u64)key << 32 | (0xFFFFFFFFu - c); }
__device__ __forceinline__ unsigned topk_index(u64 pair) { return 0xFFFFFFFFu - (unsigned)pair; }

#define TOPK_NT 256      // threads of a workgroup, or 64 where rows are short and many
#define TOPK_CAND(nt) ((nt) == 64 ? 512 : 1024)   // elements that are collected at most
#define TOPK_PAD 16      // and zeros behind them, which are below every pair
#define TOPK_LOADS 4     // pieces of 16 bytes that a thread loads at once
#define TOPK_SEGS 8      // segments of a thread: 16 take LDS from two of the 8 workgroups that a compute unit holds

#define TOPK_WAVE 4096       // elements of a row that one wave takes at most
#define TOPK_PART 4096       // elements of a part that one round of loads of fp32 takes
#define TOPK_PAIRS 4096      // pairs that a merge holds in LDS at most
#define TOPK_BLOCKS 512      // workgroups that are worth having, a row has no more parts: 300x60000 fp32, k = 50 17.6 us (with 1024 22.2)

template <int NT>
struct TopkShared {
  __attribute__((aligned(16))) u64 cand[TOPK_CAND(NT) + TOPK_PAD];   // before, the threads' maxima
  float seg[TOPK_SEGS][NT];                                          // the segments' largest; then the list of those that are read again
  unsigned hist[256];
  unsigned n, hits, bin, need, wave[NT / 64];
};

// n candidates (all different) -> the places of the k largest; out(place, pair).  The candidates are whole behind its barrier.
template <int NT, class F>
__device__ __forceinline__ void topk_place(u64* cand, int n, int k, F&& out) {
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  if (threadIdx.x < TOPK_PAD) cand[n + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const u64 mine = cand[i];
    int place = 0;
    for (int j = 0; j < n; j += TOPK_PAD) {
      u64x2 v[TOPK_PAD / 2];
#pragma unroll
      for (int u = 0; u < TOPK_PAD / 2; ++u) v[u] = *(const u64x2*)(cand + j + 2 * u);
#pragma unroll
      for (int u = 0; u < TOPK_PAD / 2; ++u) place += (v[u][0] > mine) + (v[u][1] > mine);
    }
    if (place < k) out(place, mine);
  }
}

// The k largest of C elements into sh.cand[0, k), in any order, whatever they are: the k-th largest key by four passes, 8 bits of the key
// each (a histogram of the elements that agree with the bits found so far), then the elements above it, and those equal to it by
// rising index until k are there.
template <class T, int NT>
__device__ __noinline__ void topk_radix_row(const T* __restrict__ x, int64_t C, unsigned c0, int k, TopkShared<NT>& sh) {
  const int tid = threadIdx.x;
  unsigned prefix = 0, need = (unsigned)k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) sh.hist[i] = 0;
    __syncthreads();
    for (int64_t c = tid; c < C; c += NT) {
      const unsigned key = topk_key((float)x[c]);
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned have = 0, b = 255;
      while (have + sh.hist[b] < need) have += sh.hist[b--];   // the bins below hold the rest: the sum over all of them is >= need
      sh.bin = b;
      sh.need = need - have;
    }
    __syncthreads();
    prefix = (prefix << 8) | sh.bin;
    need = sh.need;
    __syncthreads();
  }
  if (tid == 0) sh.n = 0;
  __syncthreads();
  for (int64_t c = tid; c < C; c += NT) {
    const unsigned key = topk_key((float)x[c]);
    if (key > prefix) sh.cand[atomicAdd(&sh.n, 1u)] = topk_pair(key, c0 + (unsigned)c);   // k - need of them
  }
  unsigned base = 0;
  for (int64_t cb = 0; cb < C && base < need; cb += NT) {
    const int64_t c = cb + tid;
    const bool hit = c < C && topk_key((float)x[c]) == prefix;
    const u64 ballot = __ballot(hit);
    __syncthreads();
    if ((tid & 63) == 0) sh.wave[tid >> 6] = (unsigned)__popcll(ballot);
    __syncthreads();
    unsigned before = base, all = 0;
    for (int w = 0; w < NT / 64; ++w) {
      if (w < (tid >> 6)) before += sh.wave[w];
      all += sh.wave[w];
    }
    before += (unsigned)__popcll(ballot & ((1ull << (tid & 63)) - 1));
    if (hit && before < need) sh.cand[(unsigned)k - need + before] = topk_pair(prefix, c0 + (unsigned)c);
    base += all;
  }
  __syncthreads();
}

// The largest of a piece's elements, NaN where there is one (in classes of neighbours: MX of them)
template <class T, int MX>
__device__ __forceinline__ void topk_most(const gmk_u32x4& v, float* best) {
  constexpr int VEC = gmk_elem<T>::VEC;
#pragma unroll
  for (int i = 0; i < VEC; ++i) best[i * MX / VEC] = __builtin_elementwise_maximum(best[i * MX / VEC], gmk_piece<T>(v, i));
}

// The k largest of C elements: out(place, pair).  Each thread has MX maxima, of as many classes of its elements.
template <class T, int NT, int MX, class F>
__device__ __forceinline__ void topk_row(const T* __restrict__ x, int64_t C, unsigned c0, int k, TopkShared<NT>& sh, F&& out) {
  constexpr int VEC = gmk_elem<T>::VEC;
  static_assert(MX * NT * 4 <= (int)sizeof(sh.cand), "the maxima fit");
  constexpr int64_t LOAD = (int64_t)NT * VEC, GROUP = LOAD * TOPK_LOADS;   // elements of one load of all threads; of one round of loads
  const int tid = threadIdx.x, lane = tid & 63;
  // Rounds of loads, of the row and of a segment; pieces of a segment.  A segment is a single load where there are at most two rounds:
  // 4000x10000 bf16, k = 100 33.0 us, with whole rounds 37.3.
  static_assert(TOPK_SEGS == 2 * TOPK_LOADS, "segments of up to two rounds");
  const int64_t groups = (C + GROUP - 1) / GROUP, per_seg = (groups + TOPK_SEGS - 1) / TOPK_SEGS;
  const unsigned pieces = groups <= 2 ? 1u : (unsigned)per_seg * TOPK_LOADS;
  const float low = -__builtin_inff();
  float best[MX];
#pragma unroll
  for (int i = 0; i < MX; ++i) best[i] = low;
  const int64_t e0 = (int64_t)tid * VEC;
  gmk_u32x4 v[TOPK_LOADS];   // behind the loop: the last round, which is all of a short row
  auto load = [&](int64_t h) {
    const int64_t e = e0 + h * GROUP;
    if ((h + 1) * GROUP <= C) {
#pragma unroll
      for (int i = 0; i < TOPK_LOADS; ++i) v[i] = gmk_load16(x + e + i * LOAD);
    } else {
#pragma unroll
      for (int i = 0; i < TOPK_LOADS; ++i) v[i] = gmk_row_piece(x, e + i * LOAD, C);
    }
  };
  auto close = [&](const float* mine, int64_t s) {   // segment s of this thread
    float all = mine[0];
#pragma unroll
    for (int i = 0; i < MX; ++i) {
      best[i] = __builtin_elementwise_maximum(best[i], mine[i]);
      all = __builtin_elementwise_maximum(all, mine[i]);
    }
    sh.seg[s][tid] = all;
  };
  float mine[MX];
  auto open = [&]() {
#pragma unroll
    for (int i = 0; i < MX; ++i) mine[i] = low;
  };
  if (groups <= 2) {
    for (int64_t h = 0; h < groups; ++h) {
      load(h);
#pragma unroll
      for (int i = 0; i < TOPK_LOADS; ++i) {
        open();
        topk_most<T, MX>(v[i], mine);
        close(mine, h * TOPK_LOADS + i);
      }
    }
  } else {
    for (int64_t g = 0, s = 0; g < groups; g += per_seg, ++s) {
      open();
      const int64_t end = g + per_seg < groups ? g + per_seg : groups;
      for (int64_t h = g; h < end; ++h) {
        load(h);
#pragma unroll
        for (int i = 0; i < TOPK_LOADS; ++i) topk_most<T, MX>(v[i], mine);
      }
      close(mine, s);
    }
  }
  unsigned* const maxima = (unsigned*)sh.cand;
#pragma unroll
  for (int i = 0; i < MX; ++i) maxima[i * NT + tid] = topk_key(best[i]);
  if (tid == 0) sh.n = sh.hits = 0;
  __syncthreads();
  // The k-th largest of the NT * MX maxima, its upper 18 bits (a lower bound is enough): every wave searches for itself, bit by bit.
  // A short row is collected whole.
  unsigned bound = 0;
  if (C > 64) {
    unsigned m[MX * NT / 64];
#pragma unroll
    for (int i = 0; i < MX * NT / 64; ++i) m[i] = maxima[i * 64 + lane];
    for (int bit = 31; bit >= 14; --bit) {
      const unsigned up = bound | 1u << bit;
      int have = 0;
#pragma unroll
      for (int i = 0; i < MX * NT / 64; ++i) have += __popcll(__ballot(m[i] >= up));
      if (have >= k) bound = up;
    }
  }
  const float limit = topk_value(bound);   // NaN (k maxima are) lets everything through
  unsigned again = 0;   // segments of this thread that reach it
  if (groups > 1)
    for (int i = 0; i < TOPK_SEGS; ++i)
      if ((groups == 2 || i * per_seg < groups) && !(sh.seg[i][tid] < limit)) again |= 1u << i;
  __syncthreads();
  auto collect = [&](const gmk_u32x4& v, int64_t e) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float f = gmk_piece<T>(v, i);
      if (!(f < limit) && (e + VEC <= C || e + i < C)) {
        const unsigned at = atomicAdd(&sh.n, 1u);
        if (at < TOPK_CAND(NT)) sh.cand[at] = topk_pair(topk_key(f), c0 + (unsigned)(e + i));
      }
    }
  };
  if (groups == 1) {
#pragma unroll
    for (int i = 0; i < TOPK_LOADS; ++i) collect(v[i], e0 + i * LOAD);
  } else {
    // Each of these holds an element at least that reaches the limit: a list of them that is too long means as many candidates.  Their
    // pieces are shared out among all threads, so that they are read at once and not one segment of a thread after the other.
    unsigned* const list = (unsigned*)sh.seg;
    while (again) {
      list[atomicAdd(&sh.hits, 1u)] = (unsigned)(__ffs(again) - 1) * NT + tid;
      again &= again - 1;
    }
    __syncthreads();
    const unsigned hits = sh.hits;
    if (hits > TOPK_CAND(NT)) {
      if (tid == 0) sh.n = hits;
    } else {
      const unsigned all = hits * pieces;   // < 2^29
      for (unsigned q = tid; q < all; q += NT * TOPK_LOADS) {
        gmk_u32x4 v[TOPK_LOADS];
        int64_t e[TOPK_LOADS];
#pragma unroll
        for (int i = 0; i < TOPK_LOADS; ++i) {
          const unsigned at = q + i * NT, hit = at / pieces, from = list[hit < hits ? hit : 0];
          e[i] = at < all ? (int64_t)(from % NT) * VEC + ((int64_t)(from / NT) * pieces + at % pieces) * LOAD : C;
          v[i] = gmk_row_piece(x, e[i], C);
        }
#pragma unroll
        for (int i = 0; i < TOPK_LOADS; ++i) collect(v[i], e[i]);
      }
    }
  }
  __syncthreads();
  int n = (int)sh.n;
  if (n > TOPK_CAND(NT)) {
    __syncthreads();
    topk_radix_row<T, NT>(x, C, c0, k, sh);
    n = k;
  }
  topk_place<NT>(sh.cand, n, k, out);
}

template <class T, int NT, int MX>
__global__ __launch_bounds__(NT) void topk_rows_kernel(const T* __restrict__ x, T* __restrict__ value, int* __restrict__ index,
                                                            int64_t C, int k) {
  __shared__ TopkShared<NT> sh;
  const int64_t row = blockIdx.x;
  const T* xr = x + row * C;
  topk_row<T, NT, MX>(xr, C, 0u, k, sh, [&](int place, u64 pair) {
    const unsigned c = topk_index(pair);
    value[row * k + place] = xr[c];
    index[row * k + place] = (int)c;
  });
}

// part blockIdx.x % parts of row blockIdx.x / parts -> its sorted list of k pairs
template <class T, int MX>
__global__ __launch_bounds__(TOPK_NT) void topk_parts_kernel(const T* __restrict__ x, u64* __restrict__ list, int64_t C, int k, int parts, int64_t len) {
  __shared__ TopkShared<TOPK_NT> sh;
  const int64_t row = blockIdx.x / (unsigned)parts, part = blockIdx.x % (unsigned)parts;
  const int64_t from = part * len, have = part == parts - 1 ? C - from : len;
  u64* to = list + (int64_t)blockIdx.x * k;
  topk_row<T, TOPK_NT, MX>(x + row * C + from, have, (unsigned)from, k, sh, [&](int place, u64 pair) { to[place] = pair; });
}

// One workgroup a row.  A lower bound of the k-th largest pair's key from the heads of the lists (4 k pairs, so that it is a close one
// unless a few lists hold most of the result); the pairs that reach it are collected and placed as in topk_row.  Where they do not fit, a
// pair's place is its own in its list plus, for each other list, how many of it are larger (by halving).
template <class T>
__global__ __launch_bounds__(TOPK_NT) void topk_merge_kernel(const T* __restrict__ x, const u64* __restrict__ list, T* __restrict__ value,
                                                             int* __restrict__ index, int64_t C, int k, int parts) {
  extern __shared__ u64 pairs[];
  __shared__ __attribute__((aligned(16))) u64 cand[TOPK_CAND(TOPK_NT) + TOPK_PAD];
  __shared__ unsigned s_n;
  const int64_t row = blockIdx.x;
  const int all = parts * k, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < all; i += 8 * TOPK_NT) {
    u64 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i + u * TOPK_NT < all ? list[row * all + i + u * TOPK_NT] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * TOPK_NT < all) pairs[i + u * TOPK_NT] = v[u];
  }
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  auto put = [&](int place, u64 pair) {
    const unsigned c = topk_index(pair);
    value[row * k + place] = x[row * C + c];
    index[row * k + place] = (int)c;
  };
  // head at = h * parts + p: pair h of list p
  // In registers, with a step over all of them for each bit: 4 or 14 slots of 64 heads where they hold them (5x150001 fp32, k = 50: the merge
  // 5.2 us, with all 24 slots 9.4).
  const int heads = min(k, (4 * k + parts - 1) / parts), some = heads * parts;
  unsigned bound = 0;
  auto search = [&](auto slots) {
    constexpr int SLOTS = decltype(slots)::value;
    unsigned m[SLOTS];
    int p = lane % parts, h = lane / parts;   // 64 further on: 64 % parts lists and 64 / parts places
    const int dp = 64 % parts, dh = 64 / parts;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      m[i] = h < heads ? (unsigned)(pairs[p * k + h] >> 32) : 0u;
      p += dp;
      h += dh + (p >= parts ? 1 : 0);
      p -= p >= parts ? parts : 0;
    }
    for (int bit = 31; bit >= 14; --bit) {
      const unsigned up = bound | 1u << bit;
      int have = 0;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) have += __popcll(__ballot(m[i] >= up));
      if (have >= k) bound = up;
    }
  };
  constexpr int MOST = (4 * GMK_TOPK_MAX + TOPK_BLOCKS + 63) / 64;
  if (some <= 4 * 64) search(std::integral_constant<int, 4>{});
  else if (some <= 14 * 64) search(std::integral_constant<int, 14>{});
  else search(std::integral_constant<int, MOST>{});
  for (int i = threadIdx.x; i < all; i += TOPK_NT)
    if ((unsigned)(pairs[i] >> 32) >= bound) {
      const unsigned at = atomicAdd(&s_n, 1u);
      if (at < TOPK_CAND(TOPK_NT)) cand[at] = pairs[i];
    }
  __syncthreads();
  const int n = (int)s_n;
  if (n <= TOPK_CAND(TOPK_NT)) {
    topk_place<TOPK_NT>(cand, n, k, put);
    return;
  }
  for (int i = threadIdx.x; i < all; i += TOPK_NT) {
    const u64 mine = pairs[i];
    const int own = i / k;
    int place = i - own * k;
    for (int p = 0; p < parts && place < k; ++p) {
      if (p == own) continue;
      int lo = 0, hi = k;   // pairs [0, lo) are larger, [hi, k) smaller
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pairs[p * k + mid] > mine) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
    }
    if (place < k) put(place, mine);
  }
}

// parts of a row: as many as give the card something to do, none longer than a round of loads needs where that is few enough
static int topk_parts(int64_t n, int64_t C, int k) {
  int64_t p = n < TOPK_BLOCKS ? TOPK_BLOCKS / n : 1;
  const int64_t rounds = C < 2 * TOPK_PART ? 1 : (C + TOPK_PART - 1) / TOPK_PART, fit = TOPK_PAIRS / k;
  if (p > rounds) p = rounds;
  if (p > fit) p = fit;
  return p < 2 ? 1 : (int)p;
}
// elements of all parts but the last, whole pieces of fp32; the last has at least C / parts - 4 parts > 2000 (and k <= 256)
static int64_t topk_part_len(int64_t C, int parts) { return ((C + parts - 1) / parts + 3) / 4 * 4; }

extern "C" size_t gmk_topk_rows_workspace_bytes(int64_t n, int64_t C, int k) {
  if (n <= 0 || C <= 0 || k <= 0 || k > GMK_TOPK_MAX) return 0;
  const int parts = topk_parts(n, C, k);
  return parts == 1 ? 0 : (size_t)n * parts * k * sizeof(u64);
}

extern "C" int gmk_topk_rows(const void* x, int xtype, void* value, int* index, int64_t n, int64_t C, int k, void* ws,
                             size_t ws_bytes, gmk_stream_t stream) {
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  GMK_REQUIRE(n >= 0 && C > 0 && k > 0 && k <= C, GMK_E_SHAPE);
  GMK_REQUIRE(k <= GMK_TOPK_MAX && C < 0x7FFFFFFFll, GMK_E_TOO_LARGE);
  if (n == 0) return GMK_OK;
  const int parts = topk_parts(n, C, k);
  GMK_REQUIRE(x && value && index && (ws || parts == 1), GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned_to(value, gmk_dtype_size(xtype)) &&
              gmk_aligned_to(index, 4) && (parts == 1 || gmk_aligned16(ws)), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_topk_rows_workspace_bytes(n, C, k), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_topk_rows, x, xtype, value, index, n, C, k, ws, ws_bytes, stream);
  const int64_t len = parts == 1 ? C : topk_part_len(C, parts);
  return gmk_with_dtype(xtype, [&](auto t) -> int {
    using T = decltype(t);
    const T* xt = (const T*)x;
    hipStream_t st = (hipStream_t)stream;
    // One maximum a thread where that makes at least twice k of them, else four.  A wave a row for rows of a few pieces a thread, of more
    // where the card is full of rows: 8192x1000 fp32, k = 10 13.0 us, 256 threads 22.7; 4096x4096 bf16, k = 64 16.8 (24.3), but 1024x4000 fp32,
    // k = 10 7.9 (7.3) and 256x1000 5.2 (4.7).
    const bool many = k <= TOPK_NT / 2 && len >= (int64_t)2 * k * gmk_elem<T>::VEC;
    if (parts == 1) {
      auto go = [&](auto kernel, int nt) -> int {
        GMK_REQUIRE(gmk_grid_ok(n, nt), GMK_E_TOO_LARGE);
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(nt), 0, st, xt, (T*)value, index, C, k);
        GMK_CHECK_LAUNCH();
        return GMK_OK;
      };
      if (k <= 64 && C <= (n >= 2048 ? TOPK_WAVE : TOPK_WAVE / 8)) return go(topk_rows_kernel<T, 64, 4>, 64);
      if (many) return go(topk_rows_kernel<T, TOPK_NT, 1>, TOPK_NT);
      return go(topk_rows_kernel<T, TOPK_NT, 4>, TOPK_NT);
    }
    if (many) hipLaunchKernelGGL((topk_parts_kernel<T, 1>), dim3((unsigned)(n * parts)), dim3(TOPK_NT), 0, st, xt, (u64*)ws, C, k, parts, len);
    else hipLaunchKernelGGL((topk_parts_kernel<T, 4>), dim3((unsigned)(n * parts)), dim3(TOPK_NT), 0, st, xt, (u64*)ws, C, k, parts, len);
    GMK_CHECK_LAUNCH();
    hipLaunchKernelGGL((topk_merge_kernel<T>), dim3((unsigned)n), dim3(TOPK_NT), parts * k * (int)sizeof(u64), st, xt, (const u64*)ws, (T*)value, index, C, k, parts);
    GMK_CHECK_LAUNCH();
    return GMK_OK;
  });
}
