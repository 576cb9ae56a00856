// gemm_i8.hip -- y = act((xq wq^T) * xscale * wscale + bias) on the 8-bit matrix instructions (v_mfma_i32_16x16x64_i8).  No
// counterpart in the reference: the 8-bit form of its nn.Linear (models/classifiers.py:19-20) for inference.
//
// The sum is a 32-bit integer, exact for K <= 131,056 (K * 128 * 128 < 2^31), so neither the order of K nor a split of it shows
// in the result.  The weight is the instruction's first operand: its 16 rows are the result's rows, so that a lane holds 4
// consecutive outputs of one row of y and stores them together.
#include "rows.h"
#include "quantize.h"
#include "plan.h"
#include <atomic>

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The sum's conversion rounds it to 24 bits where it is beyond 2^24, the product with the row's scale rounds, and the one with the
// column's together with the bias: three roundings of 2^-24, then the activation's and the one to the output's type.
__device__ __forceinline__ float4 i8_scaled(const i32x4& v, float xs) {
  return make_float4((float)v[0] * xs, (float)v[1] * xs, (float)v[2] * xs, (float)v[3] * xs);
}
__device__ __forceinline__ float4 i8_column(const float4& v, const float4& s, const float4& b) {
  return make_float4(fmaf(v.x, s.x, b.x), fmaf(v.y, s.y, b.y), fmaf(v.z, s.z, b.z), fmaf(v.w, s.w, b.w));
}
// a NaN stays one: a row without a scale must not look like a row of zeros
__device__ __forceinline__ float4 i8_relu(const float4& z) {
  return make_float4(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y, z.z < 0.f ? 0.f : z.z, z.w < 0.f ? 0.f : z.w);
}
template <class T>
__device__ __forceinline__ void i8_put4(const float4& z, T* p, int have) {   // the first `have` of 4 columns
  T t[4] = {(T)z.x, (T)z.y, (T)z.z, (T)z.w};
  if (have >= 4) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) p[i] = t[i];
  }
}

// All 4, past the caches, where the operands' tiles stay instead: 1053x432x29312 33.7 us (through them 35.8), 8192x4096x16384 451 to 457 (454
// to 459).  Only where rows are whole lines of 128 bytes: parts of a line that the caches do not join cost 2204x256x29857 84.7 us (45.2).
template <class T>
__device__ __forceinline__ void i8_stream4(const float4& z, T* p) {
  typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  T4 t = {(T)z.x, (T)z.y, (T)z.z, (T)z.w};
  asm volatile("");   // or the compiler makes one store of this and another branch's, without the hint
  __builtin_nontemporal_store(t, (T4*)p);
  asm volatile("");
}

// ---- tiles through LDS -------------------------------------------------------------------------------------------------------
// A workgroup of WGN x WGM waves makes tiles of BN columns times BM rows of y, one after the other.  BK bytes of K of both operands
// are staged at a time, straight from memory into LDS (16 bytes a lane, no registers), in a ring of S stages: the loads run S - 1
// chunks ahead, over the end of one tile into the next, so that they also run under a tile's epilogue; one barrier a chunk.
//
// A staged row is BK / 16 pieces of 16 bytes; piece c of row r lies at place c ^ f(r), with f so that the 8 (or 16) lanes that read
// one piece of as many consecutive rows together touch every bank once.  LDS is filled in lane order, so it is the address in memory
// that is permuted: a row's lanes still read its BK bytes in one go.
// Rows behind the last one and pieces behind K are past the buffer's end for the load, which makes them zeros.
//
// Measured, bf16 out: 8192x8192x8192 409 to 422 us, 2600 to 2690 TOP/s (a copy-free loop of the instruction reaches 4000 to 4350);
// 8192x4096x16384 450 to 457 us, with the quantiser before it 437 to 448 (its q is still in the caches).  The matrix cores are busy in 59 % (K = 4096) to
// 69 % (K = 8192) of the cycles, at the 1.9 GHz that the card holds under this load; LDS has no bank conflict.  What is left is the end of a
// tile, when all units write their 128 KB at once: 8192x1024x16384 takes 154 us of which the products are 90.
#define I8_BK 128
__device__ __forceinline__ int i8_place(int row, int piece) { return piece ^ (row & 7); }

// buffer descriptor of a wave: address, bytes, raw 32-bit format
__device__ __forceinline__ i32x4 i8_buffer(const void* base, int bytes) {
  const uint64_t p = (uint64_t)base;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)p), __builtin_amdgcn_readfirstlane((int)(unsigned)(p >> 32)),
               __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}

template <int ROWS, int NTHR>
struct I8Stage {
  static constexpr int LOADS = ROWS * 8 / NTHR, STEP = NTHR / 8;   // 16-byte pieces a thread loads for a chunk, STEP rows apart
  static_assert(LOADS * STEP == ROWS && STEP % 8 == 0, "a chunk is whole loads, a thread's pieces at one place of their rows");
  i32x4 rsrc;

  // this thread's first piece in the tile's rows, for the chunk at column k; past the buffer's end where it lies behind K
  static __device__ __forceinline__ int first(int k, int K) {
    const int row = threadIdx.x >> 3, column = i8_place(row, threadIdx.x & 7) * 16;
    return k + column < K ? row * K + column : GMK_OOB;
  }
  // `rows` rows of the tile exist (none: every load gives zeros)
  __device__ __forceinline__ void tile(const signed char* base, int row0, int rows, int K) {
    rsrc = i8_buffer(base + (int64_t)row0 * K, rows * K);   // at most 256 * 131056 bytes
  }
  // Load i of the chunk at column k into LDS, `lds` the byte address of this wave's first 64 pieces.  In asm, as the compiler would
  // wait for every load that is out before it reads LDS at all; a load to LDS has no result register, and the loop below counts it.
  // m0 is a reserved register, which no clobber list may name: the compiler keeps nothing in it and sets it where it needs it itself.
  __device__ __forceinline__ void load(int i, unsigned lds, int first, int k, int K) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"((int)lds + i * NTHR * 16), "v"(first + i * STEP * K), "s"(rsrc),
                 "s"(k) : "memory");
  }
};

template <class T, int BN, int BM, int WGN, int WGM, int S>
__global__ __launch_bounds__(64 * WGN * WGM, 2) void gemm_i8_tile_kernel(const signed char* __restrict__ xq, const float* __restrict__ xscale,
                                                                      const signed char* __restrict__ wq, const float* __restrict__ wscale,
                                                                      const float* __restrict__ bias, T* __restrict__ y, int M, int K, int N,
                                                                      int act, int tiles_m, int tiles_n) {
  constexpr int NTHR = 64 * WGN * WGM, TN = BN / WGN / 16, TM = BM / WGM / 16;
  constexpr int BUF = (BN + BM) * I8_BK, WLOADS = I8Stage<BN, NTHR>::LOADS, LOADS = WLOADS + I8Stage<BM, NTHR>::LOADS;
  extern __shared__ __attribute__((aligned(128))) signed char lds[];   // S stages of BN + BM rows, then the epilogue's part
  // The tiles of one XCD (workgroups go round the 8 of them) are neighbours: a group of 8 rows of tiles, column by column.
  const int all = tiles_m * tiles_n, xcd = blockIdx.x & 7;
  const int first = xcd * (all >> 3) + min(xcd, all & 7), last = first + (all >> 3) + (xcd < (all & 7) ? 1 : 0);
  const int step = ((int)gridDim.x - xcd + 7) >> 3;
  int tile = first + (int)(blockIdx.x >> 3);
  if (tile >= last) return;
  auto corner = [&](int t, int& m0, int& n0) {
    const int g = t / (8 * tiles_n), in = t - g * 8 * tiles_n, h = min(8, tiles_m - g * 8);
    m0 = (g * 8 + in % h) * BM;
    n0 = in / h * BN;
  };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, kq = lane >> 4;
  const int wn = (wave % WGN) * (BN / WGN), wm = (wave / WGN) * (BM / WGM);
  const int chunks = (K + I8_BK - 1) / I8_BK;

  // The loads' own place in the stream of chunks.  Behind its end they go on and give zeros, so that the loop below has one path
  // and one count of what is out.
  I8Stage<BN, NTHR> sw;
  I8Stage<BM, NTHR> sx;
  const unsigned lds0 = gmk_lds_addr(lds) + __builtin_amdgcn_readfirstlane(wave) * 1024;
  int l_tile = tile, l_chunk = 0, l_stage = 0, l_k = 0;
  auto load_tile = [&]() {
    int m0 = 0, n0 = 0;
    if (l_tile < last) corner(l_tile, m0, n0);
    sw.tile(wq, n0, l_tile < last ? min(BN, N - n0) : 0, K);
    sx.tile(xq, m0, l_tile < last ? min(BM, M - m0) : 0, K);
  };
  int l_first = I8Stage<BN, NTHR>::first(0, K);
  auto load = [&](int i) {   // load i of the chunk
    const unsigned to = lds0 + l_stage * BUF;
    if (i < WLOADS) sw.load(i, to, l_first, l_k, K);
    else sx.load(i - WLOADS, to + BN * I8_BK, l_first, l_k, K);
  };
  auto load_end = [&]() {
    l_stage = l_stage == S - 1 ? 0 : l_stage + 1;
    if (++l_chunk == chunks) {
      l_chunk = 0;
      l_tile += step;
      load_tile();
    }
    l_k = l_tile < last ? l_chunk * I8_BK : 0;   // a buffer's bytes less this column are what a load is checked against
    // only a last chunk that is not whole, and the one behind it, differ from the chunk before
    if (l_chunk == 0 || (l_chunk + 1) * I8_BK > K) l_first = I8Stage<BN, NTHR>::first(l_chunk * I8_BK, K);
  };
  load_tile();
  // Wait until at most `chunks_out` chunks of this wave's loads are out (they return in order) and its own reads of LDS are done, then
  // until every wave is here.  The first `fresh` chunks behind an epilogue are known to be there: waiting for the count would also
  // wait for the epilogue's stores.
  int fresh = 0;
  auto arrive = [&](auto chunks_out) {
    if (fresh > 0) {
      --fresh;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(chunks_out)::value * LOADS) : "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // A wave's part of LDS for its epilogue; until then it holds the tile's scales and bias, which are loaded at the tile's start:
  // XS of its rows, LS each of its columns' scales and bias (zeros where there are none).
  constexpr int LD = TN * 16, XS = (TM * 16 + 63) / 64 * 64, LS = LD < 64 ? 64 : LD;
  static_assert(XS + 2 * LS <= 16 * LD && XS % 64 == 0 && LS % 64 == 0, "the scales fit a wave's part");
  float* const part = (float*)(lds + S * BUF) + wave * 16 * LD;
  auto load_scales = [&](int m, int n) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // what the scales and the epilogue derive from it is derived there, not kept in registers
    const unsigned to = __builtin_amdgcn_readfirstlane(gmk_lds_addr(part));
    // the epilogue before this one is done with the part: a load to LDS waits for no LDS operation that is still out
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto one = [&](const float* from, int have, int most, int at) {
      const i32x4 rs = i8_buffer(from, min(max(have, 0), most) * 4);
#pragma unroll
      for (int i = 0; i < most; i += 64)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to + (at + i) * 4), "v"((lane + i) * 4), "s"(rs) : "memory");
    };
    one(xscale + m, M - m, TM * 16, 0);
    one(wscale + n, N - n, LD, XS);
    one(bias + n, bias ? N - n : 0, LD, XS + LS);
  };
  // Operands of the two halves of a chunk: one half is read from LDS while the other is multiplied, a few reads (and loads of a later
  // chunk) behind every TM multiplications, so that neither queue ever holds up the matrix cores.
  i32x4 a[2][TN], b[2][TM];
  constexpr int READS = TN + TM, RG = (READS + (TN > 1 ? TN - 2 : 0)) / (TN > 1 ? TN - 1 : 1), LG = (LOADS + TN - 1) / TN;
  const int a0 = (wn + r) * I8_BK + i8_place(r, kq) * 16, b0 = (BN + wm + r) * I8_BK + i8_place(r, kq) * 16;
  auto read = [&](int stage, auto half, int i) {   // operand i of a half; the second half's pieces are 4 places (64 bytes) across
    constexpr int h = decltype(half)::value;
    if (i < TN) a[h][i] = *(const i32x4*)(lds + stage * BUF + (h ? a0 ^ 64 : a0) + i * 16 * I8_BK);
    else b[h][i - TN] = *(const i32x4*)(lds + stage * BUF + (h ? b0 ^ 64 : b0) + (i - TN) * 16 * I8_BK);
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
#pragma unroll 1
  for (int c = 0; c < S; ++c) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(i);
    load_end();
  }
  arrive(std::integral_constant<int, S - 1>{});
  int stage = 0;
#pragma unroll
  for (int i = 0; i < READS; ++i) read(0, I0{}, i);
  for (; tile < last; tile += step) {
    int m0, n0;
    corner(tile, m0, n0);
    load_scales(m0 + wm, n0 + wn);
    i32x4 acc[TN][TM] = {};
    auto multiply = [&](auto half, auto behind) {
      constexpr int h = decltype(half)::value;
#pragma unroll
      for (int i = 0; i < TN; ++i) {
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h][i], b[h][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        behind(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int c = 0; c < chunks; ++c) {
      multiply(I0{}, [&](int g) {
#pragma unroll
        for (int i = g * RG; i < (g + 1) * RG && i < READS; ++i) read(stage, I1{}, i);
      });
      arrive(std::integral_constant<int, S - 2>{});   // the next chunk is there, and every wave has read this one
      const int next = stage == S - 1 ? 0 : stage + 1;
      multiply(I1{}, [&](int g) {
#pragma unroll
        for (int i = g * RG; i < (g + 1) * RG && i < READS; ++i) read(next, I0{}, i);
#pragma unroll
        for (int i = g * LG; i < (g + 1) * LG && i < LOADS; ++i) load(i);   // into this chunk's stage
      });
      load_end();
      stage = next;
    }
    // The sums go through LDS, 16 of a wave's rows at a time in its own part, so that y is written in whole lines.  Piece c of row q
    // lies at place c ^ q, which spreads a column over the banks.
    // Before the first store: the scales are there, and so is all that was loaded for the next tile.
    constexpr int PER_ROW = TN * 4, STEP = 64 / PER_ROW;
    static_assert(64 % PER_ROW == 0 && 16 % STEP == 0, "a wave writes whole rows");
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    fresh = S - 1;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int r = lane & 15, kq = lane >> 4;
    const int q0 = lane / PER_ROW, col = (lane % PER_ROW) * 4;
    float xs[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) xs[j] = part[16 * j + r];
    const float4 cs = *(const float4*)(part + XS + col), cb = *(const float4*)(part + XS + LS + col);
    const float es = part[XS + lane % LD], eb = part[XS + LS + lane % LD];
    asm volatile("" ::: "memory");
    const int n = n0 + wn + col;
    const bool common = act == GMK_ACT_NONE || act == GMK_ACT_RELU || act == GMK_ACT_GELU;
    const bool whole = m0 + wm + TM * 16 <= M && n0 + wn + LD <= N;
    const bool lines = (((uintptr_t)y | (uintptr_t)((int64_t)N * sizeof(T))) & 127) == 0;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int mb = m0 + wm + 16 * j;
      if (mb >= M) break;   // before the sums are written: what a wave writes to its part it also reads
#pragma unroll
      for (int i = 0; i < TN; ++i) *(float4*)(part + r * LD + (((4 * i + kq) ^ r) & (PER_ROW - 1)) * 4) = i8_scaled(acc[i][j], xs[j]);
      __builtin_amdgcn_wave_barrier();
      if (common) {
        float4 z[16 / STEP];
#pragma unroll
        for (int u = 0; u < 16 / STEP; ++u) {
          const int q = q0 + u * STEP;
          z[u] = i8_column(*(const float4*)(part + q * LD + ((lane ^ q) & (PER_ROW - 1)) * 4), cs, cb);
        }
        if (act == GMK_ACT_GELU) {
#pragma unroll
          for (int u = 0; u < 16 / STEP; ++u) {
            float4 a, d;
            gmk_gelu_fwd4(z[u], a, d);
            z[u] = a;
          }
        } else if (act == GMK_ACT_RELU) {
#pragma unroll
          for (int u = 0; u < 16 / STEP; ++u) z[u] = i8_relu(z[u]);
        }
        T* const yq = y + (int64_t)(mb + q0) * N + n;
        if (whole && lines) {
#pragma unroll
          for (int u = 0; u < 16 / STEP; ++u) i8_stream4<T>(z[u], yq + (int64_t)u * STEP * N);
        } else if (whole) {
#pragma unroll
          for (int u = 0; u < 16 / STEP; ++u) i8_put4<T>(z[u], yq + (int64_t)u * STEP * N, 4);
        } else {
#pragma unroll
          for (int u = 0; u < 16 / STEP; ++u)
            if (mb + q0 + u * STEP < M && n < N) i8_put4<T>(z[u], yq + (int64_t)u * STEP * N, N - n);
        }
      } else {   // a rarer activation: one value a lane
#pragma unroll 1
        for (int q = lane / LD; q < 16; q += 64 / LD) {
          const int e = lane % LD, m = mb + q;
          float z = fmaf(part[q * LD + (((e >> 2) ^ q) & (PER_ROW - 1)) * 4 + (e & 3)], es, eb), u = z, d;
          if (act != GMK_ACT_NONE) gmk_act_fwd(act, z, u, d);
          if (m < M && n0 + wn + e < N) y[(int64_t)m * N + n0 + wn + e] = (T)u;
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the loads behind the end still write to this workgroup's LDS
}

static int i8_cus() {   // compute units of the current device, asked once
  static std::atomic<int> cus[16];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) return 256;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <class T, int BN, int BM, int WGN, int WGM, int S>
static int gemm_i8_tile_launch(const signed char* xq, const float* xscale, const signed char* wq, const float* wscale, const float* bias,
                               T* y, int M, int K, int N, int act, hipStream_t stream) {
  const int64_t tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  GMK_REQUIRE(tm * tn < 0x7FFFFFFFll / 8, GMK_E_TOO_LARGE);
  constexpr int bytes = S * (BN + BM) * I8_BK + BN * WGM * 16 * 4;
  static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
  auto k = gemm_i8_tile_kernel<T, BN, BM, WGN, WGM, S>;
  const hipError_t e = gmk_ensure_dyn_lds((const void*)k, bytes);
  if (e != hipSuccess) return (int)e;
  const int64_t fit = (int64_t)i8_cus() * (160 * 1024 / bytes);   // workgroups that run at once
  hipLaunchKernelGGL(k, dim3((unsigned)(tm * tn < fit ? tm * tn : fit)), dim3(64 * WGN * WGM), bytes, stream, xq, xscale, wq, wscale, bias, y,
                     M, K, N, act, (int)tm, (int)tn);
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
// A workgroup makes NT * 16 columns times 16 rows of y; its waves take turns along K, 64 bytes of each row at a time straight from
// memory into the instruction's registers, U steps in flight, and their sums meet in LDS.  Rows behind the last one are read from the
// last one and never stored; behind K the weight's piece is zero.
// Bound by the weight's bytes: 1x4096x32768 bf16 30.5 us, 4.4 TB/s with the start of the launch.
// X is the rows' type: 8-bit values with xscale, or, for at most I8_FUSED_ROWS rows of floating numbers, x itself, which every workgroup
// then quantises into its LDS while its first weights are on their way: one launch instead of two.
#define I8_FUSED_ROWS 4
#define I8_FUSED_BYTES 16384   // of quantised rows in LDS: 1x4096x32768 30.5 us (two launches 41.4), 1x4096x8192 10.4 (13.3), 4x4096x32768 38.5 (41.8),
                               // 4x4096x4096 10.4 (10.0), but 3x8192x8192 would take 21.9 (19.5)
template <class T, class X, int NT, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void gemm_i8_rows_kernel(const X* __restrict__ x, const float* __restrict__ xscale,
                                                                  const signed char* __restrict__ wq, const float* __restrict__ wscale,
                                                                  const float* __restrict__ bias, T* __restrict__ y, int M, int K, int N,
                                                                  int act, int tiles_m, int Kx) {
  constexpr bool FUSED = !std::is_same<X, signed char>::value;
  __shared__ i32x4 part[WAVES * NT * 64];
  __shared__ float xs_row[I8_FUSED_ROWS];
  extern __shared__ __attribute__((aligned(16))) signed char xlds[];   // FUSED: M rows of K bytes
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, kq = lane >> 4;
  const int n0 = (int)(blockIdx.x / (unsigned)tiles_m) * NT * 16, m0 = (int)(blockIdx.x % (unsigned)tiles_m) * 16;
  const signed char* wp[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) wp[i] = wq + (int64_t)min(n0 + 16 * i + r, N - 1) * K + kq * 16;
  const signed char* xp;
  if constexpr (FUSED) xp = xlds + min(r, M - 1) * K + kq * 16;
  else xp = x + (int64_t)min(m0 + r, M - 1) * K + kq * 16;
  i32x4 acc[NT] = {};
  const int steps = (K + 63) >> 6;
  i32x4 a[U][NT], b[U];
  auto x_step = [&](int u, int s) {
    const int k = (s + u * WAVES) * 64;
    b[u] = *(const i32x4*)(xp + (k + kq * 16 < K ? k : -kq * 16));
  };
  // this wave's steps s, s + WAVES, ...; behind K zeros of the weight (the address is then the row's first one)
  auto fetch = [&](int s) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u * WAVES) * 64;
      const bool in = k + kq * 16 < K;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const i32x4 v = *(const i32x4*)(wp[i] + (in ? k : -kq * 16));
        a[u][i] = in ? v : i32x4{0, 0, 0, 0};
      }
      if constexpr (!FUSED) x_step(u, s);
    }
  };
  auto multiply = [&](int s) {
    if constexpr (FUSED) {
#pragma unroll
      for (int u = 0; u < U; ++u) x_step(u, s);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][i], b[u], acc[i], 0, 0, 0);
  };
  fetch(wave);
  if constexpr (FUSED) {
    // M rows are shared out among the waves: all to one row, half to each of two, a quarter to each of three or four
    static_assert(WAVES == 8 && I8_FUSED_ROWS == 4, "waves a row");
    constexpr int VEC = gmk_elem<X>::VEC, KEEP = 2;
    __shared__ float red[WAVES];
    const int team = M == 1 ? 8 : M == 2 ? 4 : 2, m = wave / team, stride = team * 64 * VEC;
    const int e0 = ((wave % team) * 64 + lane) * VEC;
    const X* xr = x + (int64_t)min(m, M - 1) * Kx;
    GmkMagnitude<X> mag;
    gmk_u32x4 keep[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (e0 + i * stride < Kx) keep[i] = gmk_row_piece(xr, e0 + i * stride, Kx, 0.f);
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (e0 + i * stride < Kx) mag.scan(keep[i]);
    for (int e = e0 + KEEP * stride; e < Kx; e += stride) mag.scan(gmk_row_piece(xr, e, Kx, 0.f));
    float mx = gmk_wave_max_all(mag.value());
    if (lane == 0) red[wave] = mx;
    __syncthreads();
    for (int i = m * team; i < (m + 1) * team; ++i) mx = fmaxf(mx, red[i]);
    const GmkQuant qu(mx);
    if (m < M) {
      auto put = [&](int e, const gmk_u32x4& v) {
        unsigned w[2] = {0u, 0u};
        if (e < Kx) qu.template piece<X>(v, w);
        __builtin_memcpy(xlds + m * K + e, w, VEC);
      };
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (e0 + i * stride < K) put(e0 + i * stride, keep[i]);
      for (int e = e0 + KEEP * stride; e < K; e += stride) put(e, e < Kx ? gmk_row_piece(xr, e, Kx, 0.f) : gmk_u32x4{0u, 0u, 0u, 0u});
      if (lane == 0) xs_row[m] = qu.scale();
    }
    __syncthreads();
  }
  for (int s = wave; s < steps; s += U * WAVES) {
    multiply(s);
    if (s + U * WAVES < steps) fetch(s + U * WAVES);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) part[(wave * NT + i) * 64 + lane] = acc[i];
  __syncthreads();
  for (int q = threadIdx.x; q < NT * 64; q += 64 * WAVES) {
    const int l = q & 63;
    const int m = m0 + (l & 15), n = n0 + (q >> 6) * 16 + (l >> 4) * 4;
    if (m >= M || n >= N) continue;
    const float xs = FUSED ? xs_row[FUSED ? m : 0] : xscale[m];
    float4 cs = make_float4(0.f, 0.f, 0.f, 0.f), cb = cs;
    float *sp = &cs.x, *bp = &cb.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i < N) sp[i] = wscale[n + i];
      if (bias && n + i < N) bp[i] = bias[n + i];
    }
    i32x4 v = part[q];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += part[w * NT * 64 + q];
    float4 z = i8_column(i8_scaled(v, xs), cs, cb), d;
    if (act == GMK_ACT_RELU) z = i8_relu(z);
    else GMK_WITH_ACT(act, [&](auto f) { float4 a; f(z, a, d); z = a; });
    i8_put4<T>(z, y + (int64_t)m * N + n, N - n);
  }
}

// Kx: columns of x where it is quantised here (K is then Kx rounded up to 16); else K
template <class T, class X, int NT>
static int gemm_i8_rows_launch(const X* x, const float* xscale, const signed char* wq, const float* wscale, const float* bias, T* y, int M,
                               int K, int N, int act, int Kx, hipStream_t stream) {
  const int64_t tm = (M + 15) / 16, tn = (N + NT * 16 - 1) / (NT * 16);
  GMK_REQUIRE(gmk_grid_ok(tm * tn, 512), GMK_E_TOO_LARGE);
  const int bytes = std::is_same<X, signed char>::value ? 0 : M * K;
  hipLaunchKernelGGL((gemm_i8_rows_kernel<T, X, NT, 8, 4>), dim3((unsigned)(tm * tn)), dim3(512), bytes, stream, x, xscale, wq, wscale, bias, y, M,
                     K, N, act, (int)tm, Kx);
  GMK_CHECK_LAUNCH();
  return GMK_OK;
}

static int gemm_i8_check(int M, int K, int N, int ytype, int act) {
  GMK_REQUIRE(gmk_dtype_ok(ytype) && act >= GMK_ACT_NONE && act <= GMK_ACT_SIGMOID, GMK_E_UNSUPPORTED);
  GMK_REQUIRE(M >= 0 && N > 0 && K > 0, GMK_E_SHAPE);
  GMK_REQUIRE(K <= GMK_I8_MAX_K && M <= GMK_I8_MAX_ROWS && N <= GMK_I8_MAX_ROWS, GMK_E_TOO_LARGE);   // rows and tiles are counted in 32 bits
  return GMK_OK;
}

// Which kernel: by the tiles that a shape has, as all that counts is how many of the 256 compute units work and how often each
// begins anew.  Times in us of the kernel alone on an MI355X (M x K x N, bf16 out):
//   16x16 with its waves along K: few tiles.  256x4096x256 6.0 (32x32 tiles 9.3), 1x8192x8192 14.9 (32x16 18.5), but 64x4096x4096 17.6 (9.6)
//   32x16 the same way: up to 8 rows, any number of columns, which is the form that quantises up to 4 rows by itself (1x4096x32768 bf16 30.5).
//   From 8-bit rows 64x32 tiles would be faster at these: 1x4096x32768 37.6 (29.3), 8 rows 39.5 (29.4); 24 rows 60.6 (29.9)
//   32x32 tiles: 24x8192x8192 15.6 (64x64 19.9), 64x4096x4096 9.6 (12.0); 24x4096x32768 has twice as many as run at once: 34.6 (29.9)
//   64x32 tiles: up to 32 rows.  32x4096x32768 30.1 (64x64 31.3), but 64 rows 39.5 (32.1)
//   beyond that, the least estimate of rounds * (start and end of a tile + 128-byte chunks of K * time of one), its constants
//   measured with a unit full of that kernel: 64x64 512x4096x4096 16.2 (128x128 19.4), 128x128 with 8 waves 1024x4096x4096 21.8 (29.0, two
//   workgroups of 4 waves 25.9), 128 columns by 192 rows 700x2048x7000 16.9 (21.9, 128x128 with 8 waves 22.6), 1500x4096x4096 28.1 (30.6, 37.0),
//   128x128 with 4 waves 2048x4096x4096 34.6 (40.6, 256x256 43.2), 256x256 4096x4096x4096 55.7 (67.3)
static int gemm_i8_launch(const signed char* xq, const float* xscale, const signed char* wq, const float* wscale,
                          const float* bias, void* y, int ytype, int M, int K, int N, int act, gmk_stream_t stream) {
  const int cus = i8_cus();
  auto tiles = [&](int bn, int bm) { return ((int64_t)N + bn - 1) / bn * (((int64_t)M + bm - 1) / bm); };
  const int64_t chunks = (K + I8_BK - 1) / I8_BK;
  auto estimate = [&](int bn, int bm, int at_once, float ends, float chunk) {
    return (float)((tiles(bn, bm) + at_once * cus - 1) / (at_once * cus)) * (ends + (float)chunks * chunk);
  };
  return gmk_with_dtype(ytype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto f) { return f(xq, xscale, wq, wscale, bias, (T*)y, M, K, N, act, (hipStream_t)stream); };
    if (tiles(16, 16) <= (M <= 16 ? 2 : 1) * cus)
      return gemm_i8_rows_launch<T, signed char, 1>(xq, xscale, wq, wscale, bias, (T*)y, M, K, N, act, K, (hipStream_t)stream);
    if (M <= 8) return gemm_i8_rows_launch<T, signed char, 2>(xq, xscale, wq, wscale, bias, (T*)y, M, K, N, act, K, (hipStream_t)stream);
    if (tiles(32, 32) <= 2 * cus) return go(gemm_i8_tile_launch<T, 32, 32, 2, 2, 4>);
    if (M <= 32) return go(gemm_i8_tile_launch<T, 64, 32, 2, 2, 6>);
    const float e64 = estimate(64, 64, 2, 4.f, 0.38f), e128 = estimate(128, 128, 1, 6.5f, 0.47f);
    const float e128x2 = estimate(128, 128, 2, 6.f, 0.9f), e256 = estimate(256, 256, 1, 10.f, 1.38f);
    const float e192 = estimate(128, 192, 1, 7.5f, 0.66f);
    const float least = fminf(fminf(fminf(e64, e128), fminf(e128x2, e256)), e192);
    if (least == e64) return go(gemm_i8_tile_launch<T, 64, 64, 2, 2, 4>);
    if (least == e128) return go(gemm_i8_tile_launch<T, 128, 128, 4, 2, 4>);
    if (least == e192) return go(gemm_i8_tile_launch<T, 128, 192, 4, 2, 3>);
    if (least == e128x2) return go(gemm_i8_tile_launch<T, 128, 128, 2, 2, 2>);
    return go(gemm_i8_tile_launch<T, 256, 256, 4, 2, 2>);
  });
}

extern "C" int gmk_gemm_i8(const signed char* xq, const float* xscale, const signed char* wq, const float* wscale,
                           const float* bias, void* y, int ytype, int M, int K, int N, int act, gmk_stream_t stream) {
  const int rc = gemm_i8_check(M, K, N, ytype, act);
  if (rc != GMK_OK) return rc;
  GMK_REQUIRE(K % 16 == 0, GMK_E_SHAPE);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(xq && xscale && wq && wscale && y, GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned16(xq) && gmk_aligned16(wq) && gmk_aligned_to(xscale, 4) && gmk_aligned_to(wscale, 4) &&
              gmk_aligned_to(bias, 4) && gmk_aligned_to(y, gmk_dtype_size(ytype)), GMK_E_ALIGN);
  GMK_PLAN_HOOK(gmk_gemm_i8, xq, xscale, wq, wscale, bias, y, ytype, M, K, N, act, stream);
  return gemm_i8_launch(xq, xscale, wq, wscale, bias, y, ytype, M, K, N, act, stream);
}

// few rows are quantised by the product's own workgroups
static bool linear_i8_fused(int M, int Kp) { return M <= I8_FUSED_ROWS && M * Kp <= I8_FUSED_BYTES; }

// workspace of the linear layer: the quantised rows, then their scales
static size_t linear_i8_q_bytes(int M, int K) { return (size_t)M * (size_t)((K + 15) / 16 * 16); }

extern "C" size_t gmk_linear_i8_workspace_bytes(int M, int K, int N) {
  if (M <= 0 || K <= 0 || N <= 0 || K > GMK_I8_MAX_K || linear_i8_fused(M, (K + 15) / 16 * 16)) return 0;
  return linear_i8_q_bytes(M, K) + (size_t)M * 4;
}

extern "C" int gmk_linear_i8_fwd(const void* x, int xtype, const signed char* wq, const float* wscale, const float* bias,
                                 void* y, int ytype, int M, int K, int N, int act, void* ws, size_t ws_bytes,
                                 gmk_stream_t stream) {
  const int rc = gemm_i8_check(M, K, N, ytype, act);
  if (rc != GMK_OK) return rc;
  GMK_REQUIRE(gmk_dtype_ok(xtype), GMK_E_UNSUPPORTED);
  if (M == 0) return GMK_OK;
  GMK_REQUIRE(x && wq && wscale && y && (ws || linear_i8_fused(M, (K + 15) / 16 * 16)), GMK_E_NULL);
  GMK_REQUIRE(gmk_aligned_to(x, gmk_dtype_size(xtype)) && gmk_aligned16(wq) && gmk_aligned_to(wscale, 4) &&
              gmk_aligned_to(bias, 4) && gmk_aligned_to(y, gmk_dtype_size(ytype)) && gmk_aligned16(ws), GMK_E_ALIGN);
  GMK_REQUIRE(ws_bytes >= gmk_linear_i8_workspace_bytes(M, K, N), GMK_E_WORKSPACE);
  GMK_PLAN_HOOK(gmk_linear_i8_fwd, x, xtype, wq, wscale, bias, y, ytype, M, K, N, act, ws, ws_bytes, stream);
  const int Kp = (K + 15) / 16 * 16;
  if (linear_i8_fused(M, Kp))
    return gmk_with_dtype(ytype, [&](auto t) {
      return gmk_with_dtype(xtype, [&](auto u) {
        using T = decltype(t);
        using X = decltype(u);
        if ((N + 15) / 16 <= 2 * i8_cus())
          return gemm_i8_rows_launch<T, X, 1>((const X*)x, nullptr, wq, wscale, bias, (T*)y, M, Kp, N, act, K, (hipStream_t)stream);
        return gemm_i8_rows_launch<T, X, 2>((const X*)x, nullptr, wq, wscale, bias, (T*)y, M, Kp, N, act, K, (hipStream_t)stream);
      });
    });
  signed char* q = (signed char*)ws;
  float* s = (float*)(q + linear_i8_q_bytes(M, K));
  // What the product reads again and again, q and the weight, is kept in the last cache (256 MB) by letting x pass it by, once the three
  // are about half of it: 8192x4096x16384 bf16 442 to 448 us (468 to 472), 4096x4096x16384 229 (246), but 8192x2048x8192 142.6 (137.5).
  const bool once = (int64_t)M * K * gmk_dtype_size(xtype) + (int64_t)(M + (int64_t)N) * Kp > 100 << 20;
  const int e = gmk_quantize_rows_launch(x, xtype, q, s, M, K, Kp, once, stream);
  if (e != GMK_OK) return e;
  return gemm_i8_launch(q, s, wq, wscale, bias, y, ytype, M, Kp, N, act, stream);
}
