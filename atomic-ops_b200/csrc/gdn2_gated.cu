// The diagonal gated linear recurrence over (B, L, C), forward and backward (sm_100a).
//   h_t = a_t h_{t-1} + x_t,  a_t = exp(min(g_t, 0));   a reset drops the state before its token: h_t = x_t
//   backward, from the last token to the first:  d_t = dy_t + e_t,  e_{t-1} = a_t d_t (0 at a reset),
//   dx_t = d_t,  dg_t = d_t a_t h_{t-1},  dh0 = e_{-1};  e_{L-1} is the final state's gradient.
// Past a sequence's length the state stands still and outputs and gradients are zero.
//
// The bytes bound it: x and g are read and h is written once, backward x, g and dy are read and dx and dg
// written once.  A thread walks S tokens of a channel in registers: once from zero, for what the segment
// does to a state (h -> A h + q), and, when the state that enters is known, once more as the recurrence
// itself, so that an output carries the rounding of its own steps and of the few joined segments before.
// Segments are joined over a warp's lanes by shuffles, over a CTA's warps in shared memory and over the CTAs of
// a cluster, which take neighbouring stretches of one sequence, through each other's shared memory: one launch,
// no flags in global memory, no workspace, and the same order of additions every time.  A cluster walks its
// sequence in rounds.
// The backward pass starts its segments from the states that the forward pass left at their borders (4 / S
// bytes a value) and computes h again from x: reading the rounded h instead would cost as many bytes and,
// for bf16, half a step of h in dg.
//
// Measured (forward + backward kernels): 8 x 2048 x 768 fp32 31 + 46 us, 403 MB at 5.2 TB/s; 1 x 131072 x 256
// fp32 101 + 141 us, 34 dependent rounds of 3 and 4 us; 5 x 3001 x 1001 bf16 (ragged) 48 + 80 us, rows that start
// on odd places are read two bytes at a time and the longest sequence's rounds follow one another; 16 x 3001 x 1000 bf16
// 130 + 184 us, 769 MB at 2.4 TB/s: issue slots, a value takes as many instructions as in fp32.
#include <cooperative_groups.h>
#include <cuda.h>

#include <cstring>

#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

namespace cg = cooperative_groups;

constexpr float kReset = -1.f;        // a segment's factor when a reset is in it: what entered is dropped
constexpr float kLeast = 1.40129846e-45f;  // the smallest number above zero
constexpr int kMaxWarps = 8, kMaxCluster = 8;
constexpr int kTileStages = 2;
// Tokens of a thread's segment.  Odd: where the lanes of a warp hold several segments, their rows in a tile in shared
// memory start in different banks.  Three CTAs of the backward pass fit an SM with 11, two with 15: where there are many
// sequences and channels the former count (8 x 2048 x 768: 60 -> 45 us), where few long ones are walked in clusters the
// fewer rounds (1 x 131072 x 256: 174 -> 141 us).  (bf16 channels in pairs, 5 or 7 tokens: half the loads, but the
// joins of two channels for fewer tokens: 16 x 3001 x 1000 161 + 219 us against 130 + 184.)
constexpr int tokens(bool many) { return many ? 11 : 15; }

struct GatedParams {
  const void *x, *g, *dy;
  long long xb, xl, gb, gl;           // element strides over B and L
  const float* h0;                    // (n_states, C) or null
  const int32_t* index;               // (B) or null
  const int32_t* lengths;             // (B) or null
  const uint8_t* reset;               // (B, L) or null
  void* h;                            // (B, L, C)
  float* last;                        // (B, C)
  float* marks;                       // (B, ceil(L / S), C): the state before each segment, or null
  const float* dlast;                 // (B, C) or null
  void *dx, *dg;                      // (B, L, C)
  float* dh0;                         // (B, C) or null
  uint32_t* flags;
  int B, L, C, n_states;
  int cols, clusters, lanes_log2;     // column blocks, CTAs of a cluster, lanes along C
};

__device__ __forceinline__ float value(float r) { return r; }
__device__ __forceinline__ float value(__nv_bfloat16 r) { return __bfloat162float(r); }
template <class T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
  else return v;
}
// V neighbouring channels of a step
template <class T, int V>
struct Lane;
template <>
struct Lane<float, 1> {
  using raw = float;
  static __device__ __forceinline__ void get(raw r, float* v) { v[0] = r; }
  static __device__ __forceinline__ raw put(const float* v) { return v[0]; }
};
template <>
struct Lane<__nv_bfloat16, 1> {
  using raw = __nv_bfloat16;
  static __device__ __forceinline__ void get(raw r, float* v) { v[0] = __bfloat162float(r); }
  static __device__ __forceinline__ raw put(const float* v) { return __float2bfloat16_rn(v[0]); }
};
template <>
struct Lane<__nv_bfloat16, 2> {
  using raw = __nv_bfloat162;
  static __device__ __forceinline__ void get(raw r, float* v) {
    const float2 f = __bfloat1622float2(r);
    v[0] = f.x;
    v[1] = f.y;
  }
  static __device__ __forceinline__ raw put(const float* v) { return __floats2bfloat162_rn(v[0], v[1]); }
};

// What a stretch of tokens does to the state that enters it: h -> A h + q, or q where A is kReset.  A is
// held above zero as long as no gate in the stretch is zero: an infinite state stays infinite through any number of
// them, as it does token by token.  Of a finite one at most 2^-149 is left that should not be.
struct Seg {
  float A, q;
};
__device__ __forceinline__ float step(Seg s, float h) { return s.A < 0.f ? s.q : fmaf(s.A, h, s.q); }
__device__ __forceinline__ Seg join(Seg a, Seg b) {  // a first
  Seg r;
  r.q = step(b, a.q);
  r.A = (a.A < 0.f || b.A < 0.f) ? kReset : (a.A == 0.f || b.A == 0.f) ? 0.f : fmaxf(a.A * b.A, kLeast);
  return r;
}

__device__ __forceinline__ int length_of(const GatedParams& p, int b) {
  if (!p.lengths) return p.L;
  int n = p.lengths[b];
  if (n < 0 || n > p.L) {
    if (p.flags) p.flags[1] = 1;
    n = n < 0 ? 0 : p.L;
  }
  return n;
}
__device__ __forceinline__ long long state_row(const GatedParams& p, int b) {  // -1: zeros
  if (!p.h0) return -1;
  if (!p.index) return b;
  const int i = p.index[b];
  if (i >= p.n_states) {
    if (p.flags) p.flags[1] = 1;
    return -1;
  }
  return i < 0 ? -1 : i;
}

// Bit i: token t0 + i of `live` drops the state before it.  The lanes of a segment look at a token each.
template <int S>
__device__ __forceinline__ uint32_t resets_of(const GatedParams& p, int b, long long t0, int live, int lane, int lanes) {
  if (!p.reset) return 0;
  const uint8_t* r = p.reset + b * (long long)p.L + t0;
  const int first = (threadIdx.x & 31) & ~(lanes - 1);
  uint32_t bits = 0;
  for (int i0 = 0; i0 < S; i0 += lanes) {
    const uint32_t all = __ballot_sync(0xffffffffu, i0 + lane < live && r[i0 + lane]);
    bits |= ((all >> first) & (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1u)) << i0;
  }
  return bits;
}

// The first `live` of S rows: all at once where there are S.
template <int S, class T>
__device__ __forceinline__ void rows_of(T r[S], const T* p, long long ld, int live) {
  if (live == S) {
#pragma unroll
    for (int i = 0; i < S; ++i) r[i] = __ldg(p + i * ld);
  } else {
    for (int i = 0; i < S; ++i) r[i] = T{};
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < live) r[i] = __ldg(p + i * ld);
  }
}

struct Shared {
  Seg part[2][kMaxWarps][32];       // a warp's segments together, by channel of a row of lanes, for two rounds
  Seg inbox[2][kMaxCluster][32];    // the CTAs' of the cluster, for two rounds
  uint64_t bar[2];                      // that they are there
  uint64_t full[kTileStages];           // that a stage's tiles are
  volatile int dead;                    // a wait ran out
};

// The CTAs of a cluster write what their segments come to into each other's inbox, and each write is counted at the
// receiver's barrier.  (A barrier over the cluster would order all of the CTA's memory accesses, the outputs' of the
// round before among them: 5.0 us a round of 8 CTAs.)  A CTA sends round r + 2 after it has seen every CTA's
// round r + 1, which these send after they have read round r: two boxes are enough.
__device__ __forceinline__ void send(Shared& sm, int box, int from, int to, int at, Seg s) {
  uint32_t dst, bar;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(&sm.inbox[box][from][at])), "r"(to));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&sm.bar[box])), "r"(to));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(dst),
               "r"(__float_as_uint(s.A)), "r"(__float_as_uint(s.q)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  for (uint32_t it = 0;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 255u) == 255u && clock64() - t0 > kWaitCycles) return false;
  }
}

__device__ __forceinline__ void begin(Shared& sm, int n, bool tiles) {
  if (n == 1 && !tiles) return;
  if (threadIdx.x == 0) {
    mbar_init(&sm.bar[0], 1);
    mbar_init(&sm.bar[1], 1);
    for (int i = 0; i < kTileStages; ++i) mbar_init(&sm.full[i], 1);
    sm.dead = 0;
    fence_mbar_init();
  }
  if (n > 1) cg::this_cluster().sync();
  else __syncthreads();
}
__device__ __forceinline__ void tile_wait(Shared& sm, int stage, uint32_t parity, uint32_t* flags) {
  if (sm.dead || cluster_wait(&sm.full[stage], parity)) return;
  sm.dead = 1;
  if (flags) flags[2] = 1;
}
// Before the CTA ends: its copies out of shared memory are over, and had a wait run out, those into it are given time.
__device__ __forceinline__ void tiles_done(const Shared& sm) {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (sm.dead) {
    const long long t0 = clock64();
    while (clock64() - t0 < 20 * 1000 * 1000) __nanosleep(1000);
  }
}

// join() and step() where no reset and no gate of zero is about (plain), or with them.
template <bool PLAIN>
__device__ __forceinline__ Seg join_as(Seg a, Seg b) {
  if constexpr (PLAIN) return {fmaxf(a.A * b.A, kLeast), fmaf(b.A, a.q, b.q)};
  else return join(a, b);
}
template <bool PLAIN>
__device__ __forceinline__ float step_as(Seg s, float h) {
  if constexpr (PLAIN) return fmaf(s.A, h, s.q);
  else return step(s, h);
}
template <bool PLAIN>
__device__ __forceinline__ void join_warp(Seg (*part)[32], Seg all, int lanes, Seg& before) {
  const int at = threadIdx.x & 31, lane = at & (lanes - 1), warp = threadIdx.x >> 5;
  for (int d = lanes; d < 32; d <<= 1) {
    const Seg left = {__shfl_up_sync(0xffffffffu, all.A, d), __shfl_up_sync(0xffffffffu, all.q, d)};
    if (at >= d) all = join_as<PLAIN>(left, all);
  }
  if (at >= 32 - lanes) part[warp][lane] = all;
  before = {1.f, 0.f};
  if (lanes < 32) {
    before = {__shfl_up_sync(0xffffffffu, all.A, lanes), __shfl_up_sync(0xffffffffu, all.q, lanes)};
    if (at < lanes) before = {1.f, 0.f};
  }
}
template <bool PLAIN>
__device__ __forceinline__ void join_cta(Shared& sm, int round, int lanes, int rank, int n, Seg& before, float& enter, float& mine_in) {
  const int at = threadIdx.x & 31, lane = at & (lanes - 1), warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (n > 1) {
    Seg pre = {1.f, 0.f};
    for (int i = 0; i < warp; ++i) pre = join_as<PLAIN>(pre, sm.part[round & 1][i][lane]);
    if (warp == warps - 1 && at < lanes) {
      const Seg all = join_as<PLAIN>(pre, sm.part[round & 1][warp][lane]);
      for (int r = 0; r < n; ++r) send(sm, round & 1, rank, r, lane, all);
    }
    before = join_as<PLAIN>(pre, before);
  } else {                              // the state itself goes from warp to warp
    float h = enter, in = h;
    for (int i = 0; i < warps; ++i) {
      if (i == warp) in = h;
      h = step_as<PLAIN>(sm.part[round & 1][i][lane], h);
    }
    mine_in = step_as<PLAIN>(before, in);
    enter = h;
  }
}

// Joins the segments of all threads.  The lanes of a warp hold 32 / lanes neighbouring segments of the same
// channels, the warps of a CTA and the CTAs of a cluster follow one another.  `enter` is the state that the
// cluster's first segment enters with; on return `mine_in` is what this thread's enters with, and `enter` what the
// next round's first one does.  `plain`: no reset and no gate of zero in this thread's segment.
__device__ __forceinline__ void exchange(Shared& sm, int round, Seg mine, bool plain, int lanes, int rank, int n,
                                         float& enter, float& mine_in, uint32_t* flags) {
  const int lane = threadIdx.x & (lanes - 1);
  Seg before;                           // of this warp's segments before this thread's
  if (__all_sync(0xffffffffu, plain)) join_warp<true>(sm.part[round & 1], mine, lanes, before);
  else join_warp<false>(sm.part[round & 1], mine, lanes, before);
  if (__syncthreads_and(plain)) join_cta<true>(sm, round, lanes, rank, n, before, enter, mine_in);
  else join_cta<false>(sm, round, lanes, rank, n, before, enter, mine_in);
  if (n > 1) {
    Seg(*inbox)[32] = sm.inbox[round & 1];
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&sm.bar[round & 1], (uint32_t)(n * lanes * sizeof(Seg)));
    if (!sm.dead && !cluster_wait(&sm.bar[round & 1], (round >> 1) & 1)) {
      sm.dead = 1;
      if (flags) flags[2] = 1;
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      if (r < n) {
        if (r == rank) mine_in = step(before, enter);
        enter = step(inbox[r][lane], enter);
      }
  }
}

__device__ __forceinline__ float at_most_zero(float g) {  // a NaN stays one
  float r;
  asm("min.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(g));
  return r;
}
// What S tokens do to a state, from the product of their gates and the state that they make of zero.
template <int S>
__device__ __forceinline__ Seg segment(const float a[S], float A, float q, uint32_t resets, bool& plain) {
  if (resets) A = kReset;
  else if (!(A > 0.f)) {                // underflow, or a gate that is zero (or a NaN)
    bool zero = false;
#pragma unroll
    for (int i = 0; i < S; ++i) zero |= a[i] == 0.f;
    A = A != A ? A : zero ? 0.f : kLeast;
  }
  plain = plain && A > 0.f;
  return {A, q};
}

// A tile in shared memory: `tokens` rows of the lanes' 4-byte words, brought and taken away by tiled copies.  Rows past
// the sequences' end arrive as zeros (gates of one, nothing added) and are not taken away.
struct Tiles {
  CUtensorMap x, g, dy, o0, o1;         // o0: h or dx, o1: dg
  int boxes;                            // copies of a tile: their boxes have up to 256 rows
};
__host__ __device__ __forceinline__ uint32_t tile_pitch(uint32_t bytes) { return (bytes + 127) / 128 * 128; }
struct Ring {
  uint64_t* bar;
  uint8_t* base;
  uint32_t bytes;                       // of a tile
  int arrays;                           // tiles of a stage
  __device__ __forceinline__ uint32_t tile() const { return tile_pitch(bytes); }
  __device__ __forceinline__ uint32_t at(int stage, int array) const { return smem_u32(base) + (stage * arrays + array) * tile(); }
};
__device__ __forceinline__ void tile_in(uint32_t dst, const CUtensorMap* m, int c, int t, int b, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(m), "r"(c), "r"(t), "r"(b), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tile_out(const CUtensorMap* m, uint32_t src, int c, int t, int b) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(m), "r"(c), "r"(t), "r"(b),
               "r"(src)
               : "memory");
}
__device__ __forceinline__ void tiles_read() {  // what was sent away has been read from shared memory
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void stage_in(const Ring& r, const Tiles& m, int stage, int c, int t, int b, int rows) {
  mbar_arrive_expect_tx(&r.bar[stage], r.bytes * r.arrays);
  const uint32_t bar = smem_u32(&r.bar[stage]), part = r.bytes / m.boxes;
  for (int i = 0; i < m.boxes; ++i) {
    tile_in(r.at(stage, 0) + i * part, &m.x, c, t + i * rows, b, bar);
    tile_in(r.at(stage, 1) + i * part, &m.g, c, t + i * rows, b, bar);
    if (r.arrays == 3) tile_in(r.at(stage, 2) + i * part, &m.dy, c, t + i * rows, b, bar);
  }
}
template <class T>
__device__ __forceinline__ T word(uint32_t at) {
  T r;
  if constexpr (sizeof(T) == 4) {
    uint32_t u;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u) : "r"(at));
    memcpy(&r, &u, 4);
  } else {
    uint16_t u;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(u) : "r"(at));
    memcpy(&r, &u, 2);
  }
  return r;
}
template <class T>
__device__ __forceinline__ void put_word(uint32_t at, T r) {
  if constexpr (sizeof(T) == 4) {
    uint32_t u;
    memcpy(&u, &r, 4);
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(u) : "memory");
  } else {
    uint16_t u;
    memcpy(&u, &r, 2);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(u) : "memory");
  }
}

// Tiles past a sequence's length: zeros, and nothing else to do.
template <class T, int S>
__device__ __forceinline__ void zero_rows(void* out, const GatedParams& p, int b, int c, int TT, int count, int rank, int place) {
  for (long long tile = count + (rank - count % p.clusters + p.clusters) % p.clusters; tile * TT < p.L; tile += p.clusters) {
    const long long t0 = tile * TT + place * S;
    T* to = static_cast<T*>(out) + ((long long)b * p.L + t0) * p.C + c;
    for (int i = 0; i < S && t0 + i < p.L; ++i) to[i * (long long)p.C] = rounded<T>(0.f);
  }
}

// TILE: the rows come and go by tiled copies, a stage ahead of the work; else each thread reads and writes its own.
// (8 x 2048 x 768 fp32: 46 instructions a value without tiles, 41 with them, and 92 against 76 us both ways: the
// exponential is 8 of them, the segments' joins about 10.)
template <class T, int S, bool TILE>
__global__ void __launch_bounds__(32 * kMaxWarps, 3) gated_fwd_kernel(const __grid_constant__ GatedParams p,
                                                                      const __grid_constant__ Tiles m) {
  extern __shared__ __align__(128) uint8_t tiles[];
  __shared__ Shared sm;
  const int lanes = 1 << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int place = threadIdx.x >> p.lanes_log2, places = blockDim.x >> p.lanes_log2;
  const int rank = blockIdx.x % p.clusters, block = blockIdx.x / p.clusters;
  const int b = block / p.cols, c0 = (block % p.cols) * lanes, c = c0 + lane;
  const bool on = c < p.C;
  const int len = length_of(p, b);
  const long long row = state_row(p, b);
  const int segs = (p.L + S - 1) / S, TT = places * S, count = (len + TT - 1) / TT;  // tiles of TT tokens with work
  const Ring ring{sm.full, tiles, (uint32_t)(TT * lanes * sizeof(T)), 2};
  begin(sm, p.clusters, TILE);
  if (TILE && threadIdx.x == 0)
    for (int s = 0; s < kTileStages && s * p.clusters + rank < count; ++s)
      stage_in(ring, m, s, c0, (s * p.clusters + rank) * TT, b, TT / m.boxes);
  float enter = on && row >= 0 ? p.h0[row * p.C + c] : 0.f;
  float top = -1.f;                     // the largest gate
  for (int round = 0; round * p.clusters < count; ++round) {
    const int tile = round * p.clusters + rank, seg = tile * places + place, slot = round % kTileStages;
    const long long t0 = (long long)seg * S;
    const int alive = max(0, min(S, (int)min((long long)S, len - t0))), live = on ? alive : 0;
    const uint32_t words = ring.at(slot, 0) + (place * S * lanes + lane) * (int)sizeof(T);
    float a[S], q[S];
    if constexpr (TILE) {
      if (threadIdx.x == 0 && round > 0) {  // the stage of the round before takes the next one
        tiles_read();
        const int next = tile + (kTileStages - 1) * p.clusters;
        if (next < count) stage_in(ring, m, (round - 1) % kTileStages, c0, next * TT, b, TT / m.boxes);
      }
      if (tile < count) tile_wait(sm, slot, (round / kTileStages) & 1, p.flags);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        q[i] = value(word<T>(words + i * lanes * (int)sizeof(T)));
        a[i] = value(word<T>(words + ring.tile() + i * lanes * (int)sizeof(T)));
      }
      if (live < S) {                   // past the length: whatever is there
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (i >= live) q[i] = a[i] = 0.f;
      }
    } else {
      T rx[S], rg[S];
      rows_of<S>(rx, static_cast<const T*>(p.x) + b * p.xb + c + t0 * p.xl, p.xl, live);
      rows_of<S>(rg, static_cast<const T*>(p.g) + b * p.gb + c + t0 * p.gl, p.gl, live);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        q[i] = value(rx[i]);
        a[i] = value(rg[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
      top = fmaxf(top, a[i]);
      a[i] = expf(at_most_zero(a[i]));
    }
    const uint32_t resets = resets_of<S>(p, b, t0, alive, lane, lanes);
    float A = 1.f, s = 0.f, mine_in;
    bool plain = true;
    if (!resets) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        s = fmaf(a[i], s, q[i]);
        A *= a[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < S; ++i) s = ((resets >> i) & 1u) ? q[i] : fmaf(a[i], s, q[i]);
    }
    const Seg mine = segment<S>(a, A, s, resets, plain);
    exchange(sm, round, mine, plain, lanes, rank, p.clusters, enter, mine_in, p.flags);
    if (p.marks && live) p.marks[((long long)b * segs + seg) * p.C + c] = mine_in;
    const bool whole = live == S && !resets;
    T* ph = static_cast<T*>(p.h) + ((long long)b * p.L + t0) * p.C + c;
    const int rows = on && tile < count ? (int)max(0ll, min((long long)S, p.L - t0)) : 0;
    auto put = [&](int i, float y) {
      if constexpr (TILE) put_word(words + i * lanes * (int)sizeof(T), rounded<T>(y));
      else if (i < rows) ph[i * (long long)p.C] = rounded<T>(y);
    };
    if (whole) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        mine_in = fmaf(a[i], mine_in, q[i]);
        put(i, mine_in);
      }
    } else {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        mine_in = ((resets >> i) & 1u) ? q[i] : fmaf(a[i], mine_in, q[i]);
        put(i, i < live ? mine_in : 0.f);
      }
    }
    if constexpr (TILE) {
      fence_async_smem();
      __syncthreads();
      if (threadIdx.x == 0 && tile < count) {
        for (int i = 0; i < m.boxes; ++i)
          tile_out(&m.o0, ring.at(slot, 0) + i * (ring.bytes / m.boxes), c0, tile * TT + i * (TT / m.boxes), b);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  }
  if (on) zero_rows<T, S>(p.h, p, b, c, TT, count, rank, place);
  if (on && rank == 0 && place == 0) p.last[(long long)b * p.C + c] = enter;
  if (top > 0.f) p.flags[0] = 1;
  if (TILE && threadIdx.x == 0) tiles_done(sm);
  if (p.clusters > 1) cg::this_cluster().sync();  // a CTA's shared memory is written until here
}

// The tiles and segments of a sequence in reverse: round 0 has the last ones.
template <class T, int S, bool TILE>
__global__ void __launch_bounds__(32 * kMaxWarps, S < 12 ? 3 : 2) gated_bwd_kernel(const __grid_constant__ GatedParams p,
                                                                      const __grid_constant__ Tiles m) {
  extern __shared__ __align__(128) uint8_t tiles[];
  __shared__ Shared sm;
  const int lanes = 1 << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int places = blockDim.x >> p.lanes_log2, place = places - 1 - (threadIdx.x >> p.lanes_log2);
  const int rank = blockIdx.x % p.clusters, block = blockIdx.x / p.clusters;
  const int b = block / p.cols, c0 = (block % p.cols) * lanes, c = c0 + lane;
  const bool on = c < p.C;
  const int len = length_of(p, b);
  const int segs = (p.L + S - 1) / S, TT = places * S, count = (len + TT - 1) / TT;  // tiles of TT tokens with work
  const Ring ring{sm.full, tiles, (uint32_t)(TT * lanes * sizeof(T)), 3};
  begin(sm, p.clusters, TILE);
  if (TILE && threadIdx.x == 0)
    for (int s = 0; s < kTileStages && s * p.clusters + rank < count; ++s)
      stage_in(ring, m, s, c0, (count - 1 - s * p.clusters - rank) * TT, b, TT / m.boxes);
  float enter = on && p.dlast ? p.dlast[(long long)b * p.C + c] : 0.f;  // e after the last token of a round
  const T* g = static_cast<const T*>(p.g) + b * p.gb + c;
  const long long at = (long long)b * p.L * p.C + c, row = p.C;
  for (int round = 0; round * p.clusters < count; ++round) {
    const int tile = count - 1 - round * p.clusters - rank, slot = round % kTileStages;  // below 0: none
    const int seg = tile * places + place;
    const long long t0 = (long long)seg * S;
    const int alive = tile < 0 ? 0 : max(0, min(S, (int)min((long long)S, len - t0))), live = on ? alive : 0;
    const uint32_t words = ring.at(slot, 0) + (place * S * lanes + lane) * (int)sizeof(T);
    float a[S], h[S], d[S], top = -1.f;
    if constexpr (TILE) {
      if (threadIdx.x == 0 && round > 0) {  // the stage of the round before takes the next one
        tiles_read();
        const int next = tile - (kTileStages - 1) * p.clusters;
        if (next >= 0) stage_in(ring, m, (round - 1) % kTileStages, c0, next * TT, b, TT / m.boxes);
      }
      if (tile >= 0) tile_wait(sm, slot, (round / kTileStages) & 1, p.flags);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        h[i] = value(word<T>(words + i * lanes * (int)sizeof(T)));
        a[i] = value(word<T>(words + ring.tile() + i * lanes * (int)sizeof(T)));
        d[i] = value(word<T>(words + 2 * ring.tile() + i * lanes * (int)sizeof(T)));
      }
      if (live < S) {                   // past the length: whatever is there
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (i >= live) h[i] = a[i] = d[i] = 0.f;
      }
    } else {
      T rx[S], rg[S], ry[S];
      rows_of<S>(rx, static_cast<const T*>(p.x) + b * p.xb + c + t0 * p.xl, p.xl, live);
      rows_of<S>(rg, g + t0 * p.gl, p.gl, live);
      rows_of<S>(ry, static_cast<const T*>(p.dy) + at + t0 * row, row, live);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        h[i] = value(rx[i]);
        a[i] = value(rg[i]);
        d[i] = value(ry[i]);
      }
    }
    const uint32_t resets = resets_of<S>(p, b, t0, alive, lane, lanes);
    bool plain = true;
    float s = live ? p.marks[((long long)b * segs + seg) * p.C + c] : 0.f, A = 1.f, back = 0.f, e;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      top = fmaxf(top, a[i]);
      a[i] = expf(at_most_zero(a[i]));
    }
    if (!resets) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const float x = h[i];
        h[i] = s;                       // the state before the token
        s = fmaf(a[i], s, x);
      }
#pragma unroll
      for (int i = S - 1; i >= 0; --i) {
        back = a[i] * (d[i] + back);
        A *= a[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const float x = h[i];
        h[i] = s;
        s = ((resets >> i) & 1u) ? x : fmaf(a[i], s, x);
      }
#pragma unroll
      for (int i = S - 1; i >= 0; --i) back = ((resets >> i) & 1u) ? 0.f : a[i] * (d[i] + back);
    }
    const Seg mine = segment<S>(a, A, back, resets, plain);
    exchange(sm, round, mine, plain, lanes, rank, p.clusters, enter, e, p.flags);
    T* qx = static_cast<T*>(p.dx) + at + t0 * row;
    T* qg = static_cast<T*>(p.dg) + at + t0 * row;
    const int rows = on && tile >= 0 ? (int)max(0ll, min((long long)S, p.L - t0)) : 0;
    auto put = [&](int i, float ox, float og) {
      if constexpr (TILE) {
        put_word(words + i * lanes * (int)sizeof(T), rounded<T>(ox));
        put_word(words + ring.tile() + i * lanes * (int)sizeof(T), rounded<T>(og));
      } else if (i < rows) {
        qx[i * row] = rounded<T>(ox);
        qg[i * row] = rounded<T>(og);
      }
    };
    if (live == S && !resets && !(top > 0.f)) {
#pragma unroll
      for (int i = S - 1; i >= 0; --i) {
        const float ox = d[i] + e;
        e = a[i] * ox;
        put(i, ox, e * h[i]);
      }
    } else {
#pragma unroll
      for (int i = S - 1; i >= 0; --i) {
        float ox = 0.f, og = 0.f;
        if (i < live) {
          const bool r = (resets >> i) & 1u;
          ox = d[i] + e;
          e = r ? 0.f : a[i] * ox;
          og = r || value(g[(t0 + i) * p.gl]) > 0.f ? 0.f : e * h[i];
        }
        put(i, ox, og);
      }
    }
    if constexpr (TILE) {
      fence_async_smem();
      __syncthreads();
      if (threadIdx.x == 0 && tile >= 0) {
        for (int i = 0; i < m.boxes; ++i) {
          const uint32_t part = i * (ring.bytes / m.boxes);
          tile_out(&m.o0, ring.at(slot, 0) + part, c0, tile * TT + i * (TT / m.boxes), b);
          tile_out(&m.o1, ring.at(slot, 1) + part, c0, tile * TT + i * (TT / m.boxes), b);
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  }
  if (on) {
    zero_rows<T, S>(p.dx, p, b, c, TT, count, rank, place);
    zero_rows<T, S>(p.dg, p, b, c, TT, count, rank, place);
  }
  if (p.dh0 && on && rank == 0 && place == places - 1) p.dh0[(long long)b * p.C + c] = enter;
  if (TILE && threadIdx.x == 0) tiles_done(sm);
  if (p.clusters > 1) cg::this_cluster().sync();  // a CTA's shared memory is written until here
}

// A few tokens while a model answers: a thread walks them for V channels of a sequence (256 x 1 x 768 fp32: 3.1 us,
// all of it latency; the call takes 6.6).
template <class T, int V>
__global__ void __launch_bounds__(128) gated_step_kernel(const __grid_constant__ GatedParams p) {
  using L = Lane<T, V>;
  using raw = typename L::raw;
  const long long per = (p.C + V - 1) / V, i = blockIdx.x * 128ll + threadIdx.x;
  if (i >= p.B * per) return;
  const int b = (int)(i / per), c = (int)(i % per) * V;
  const int len = length_of(p, b);
  const long long row = state_row(p, b);
  float s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = row >= 0 ? p.h0[row * p.C + c + v] : 0.f;
  bool positive = false;
  for (int t = 0; t < p.L; ++t) {
    float a[V], q[V], y[V];
    const bool live = t < len;
    if (live) {
      L::get(reinterpret_cast<const raw*>(static_cast<const T*>(p.x) + b * p.xb + t * p.xl + c)[0], q);
      L::get(reinterpret_cast<const raw*>(static_cast<const T*>(p.g) + b * p.gb + t * p.gl + c)[0], a);
      const bool r = p.reset && p.reset[b * (long long)p.L + t];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        positive |= a[v] > 0.f;
        s[v] = r ? q[v] : fmaf(expf(a[v] > 0.f ? 0.f : a[v]), s[v], q[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = live ? s[v] : 0.f;
    reinterpret_cast<raw*>(static_cast<T*>(p.h) + ((long long)b * p.L + t) * p.C + c)[0] = L::put(y);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) p.last[(long long)b * p.C + c + v] = s[v];
  if (positive && p.flags) p.flags[0] = 1;
}

// ---- host ---------------------------------------------------------------------------------------
constexpr int kStepTokens = 4;

// Two channels to a lane where bf16 rows allow 4-byte accesses.
bool pairs(const gdn2_gated_desc* d) {
  return d->dtype == GDN2_BF16 && d->C % 2 == 0 && d->x_stride[0] % 2 == 0 && d->x_stride[1] % 2 == 0 &&
         d->g_stride[0] % 2 == 0 && d->g_stride[1] % 2 == 0;
}

gdn2_status check_gated(const gdn2_gated_desc* d) {
  if (!d || d->B < 1 || d->L < 0 || d->C < 1 || d->n_states < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 2; ++i)
    if (d->x_stride[i] < 0 || d->g_stride[i] < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->L > 1 << 30 || d->C > 1 << 30) return GDN2_ERR_UNSUPPORTED;
  if ((long long)d->B * ((d->C + 7) / 8) > (1ll << 27)) return GDN2_ERR_UNSUPPORTED;  // CTAs of a grid
  return GDN2_OK;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// (B, L, C) with rows `sl` and sequences `sb` elements apart, in boxes of `rows` tokens by `width` channels.  False
// where tiled copies cannot read it.
bool tile_map(CUtensorMap* map, const void* p, bool bf16, const GatedParams& q, long long sb, long long sl, int width, int rows) {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) == cudaSuccess &&
                   r == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeFn>(f)
               : nullptr;
  }();
  const long long el = bf16 ? 2 : 4;
  if (q.L == 1) sl = q.C;
  if (q.B == 1) sb = sl * q.L;
  sl = (q.L == 1 ? (sl * el + 15) / 16 * 16 : sl * el);
  sb = (q.B == 1 ? (sb * el + 15) / 16 * 16 : sb * el);
  if (!fn || reinterpret_cast<uintptr_t>(p) % 16 || sl % 16 || sb % 16 || sl <= 0 || sb <= 0 || sl >= 1ll << 40 || sb >= 1ll << 40)
    return false;
  const cuuint64_t dims[3] = {(cuuint64_t)q.C, (cuuint64_t)q.L, (cuuint64_t)q.B};
  const cuuint64_t strides[2] = {(cuuint64_t)sl, (cuuint64_t)sb};
  const cuuint32_t box[3] = {(cuuint32_t)width, (cuuint32_t)rows, 1}, unit[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(p), dims,
              strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  return encode() || (bind_context(), encode());
}

template <class T, int S>
cudaError_t launch_gated_as(bool back, GatedParams& p, cudaStream_t st) {
  constexpr bool kBf16 = sizeof(T) == 2;
  const int segs = (p.L + S - 1) / S;
  // Enough CTAs for two on every SM: narrower ones first (32-byte rows of 8 lanes, which then take more segments), then
  // clusters (forward + backward of 1 x 131072 x 256: 794 us with 64 CTAs of 32 channels in clusters of 8, 459 with
  // 128 of 16, 300 with 256 of 8; 8 x 2048 x 768: 110 us with 192 of 32, 92 with 384 of 16, 136 with 384 of 32 in
  // pairs; all before the tiles).
  int lanes_log2 = 5, clusters = 1;
  auto cols = [&] { return (int)((p.C + (1ll << lanes_log2) - 1) >> lanes_log2); };
  auto groups = [&] { return 32 >> lanes_log2; };
  while (lanes_log2 > 3 && (long long)p.B * cols() < 296 && 2 * groups() <= segs) --lanes_log2;
  int warps = (segs + groups() - 1) / groups();
  warps = warps < 1 ? 1 : warps > kMaxWarps ? kMaxWarps : warps;
  constexpr int kEven = 8 / sizeof(T);
  if (warps * groups() * S > 256) warps = (warps + kEven - 1) / kEven * kEven;  // two boxes of a tile, each on 128 bytes
  const int places = warps * groups(), TT = places * S;
  // The same with lengths, whatever part of the tiles may be empty: over 156 shapes (2 to 24 sequences of 1500 to 8192 tokens,
  // 256 to 1536 channels, both types) a doubling beyond this takes 1 to 37 % longer in all but a few, full sequences and
  // such of any length alike (up to 700 CTAs: 8 % longer on average; 5 x 3001 x 1001 bf16 104 -> 85 us with some lengths, 112
  // -> 126 with others, 4 x 4096 x 512 fp32 57 -> 66, 8 x 2048 x 256 35 -> 45).
  while (clusters < kMaxCluster && (long long)p.B * cols() * clusters * 2 <= 296 && clusters * places < segs) clusters *= 2;
  p.cols = cols();
  p.clusters = clusters;
  p.lanes_log2 = lanes_log2;
  Tiles m;
  m.boxes = TT > 256 ? 2 : 1;
  const int width = 1 << lanes_log2, rows = TT / m.boxes;
  const long long cb = (long long)p.L * p.C, cl = p.C;
  bool tile = p.L > 0 && tile_map(&m.x, p.x, kBf16, p, p.xb, p.xl, width, rows) &&
              tile_map(&m.g, p.g, kBf16, p, p.gb, p.gl, width, rows) &&
              tile_map(&m.o0, back ? p.dx : p.h, kBf16, p, cb, cl, width, rows);
  if (tile && back)
    tile = tile_map(&m.dy, p.dy, kBf16, p, cb, cl, width, rows) && tile_map(&m.o1, p.dg, kBf16, p, cb, cl, width, rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.cols * clusters));
  cfg.blockDim = dim3(32u * warps);
  cfg.dynamicSmemBytes = tile ? (size_t)kTileStages * (back ? 3 : 2) * tile_pitch(TT * (uint32_t)sizeof(T) * width) : 0;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)clusters;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto go = [&](auto kernel, unsigned long long& done) {
    if (cfg.dynamicSmemBytes > 32768) {
      const cudaError_t e = smem_attr_once(kernel, kTileStages * 3 * kMaxWarps * tokens(false) * 32 * 4, done);
      if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, p, m);
  };
  static unsigned long long done[2] = {};
  if (tile) return back ? go(gated_bwd_kernel<T, S, true>, done[1]) : go(gated_fwd_kernel<T, S, true>, done[0]);
  return back ? go(gated_bwd_kernel<T, S, false>, done[1]) : go(gated_fwd_kernel<T, S, false>, done[0]);
}

// Enough channels for more than one CTA of 16 lanes on every SM's two places.
bool many(long long B, long long C) { return B * ((C + 15) / 16) >= 296; }
template <class T>
cudaError_t launch_gated(bool back, GatedParams& p, cudaStream_t st) {
  return many(p.B, p.C) ? launch_gated_as<T, tokens(true)>(back, p, st) : launch_gated_as<T, tokens(false)>(back, p, st);
}

GatedParams params_of(const gdn2_gated_desc* d) {
  GatedParams p{};
  p.B = d->B; p.L = d->L; p.C = d->C; p.n_states = d->n_states;
  p.xb = d->x_stride[0]; p.xl = d->x_stride[1];
  p.gb = d->g_stride[0]; p.gl = d->g_stride[1];
  return p;
}
bool off(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
size_t access(const gdn2_gated_desc* d) { return d->dtype == GDN2_F32 || pairs(d) ? 4 : 2; }

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_gated_marks_bytes(const gdn2_gated_desc* d) {
  using namespace gdn2;
  if (check_gated(d) != GDN2_OK) return 0;
  const long long S = tokens(many(d->B, d->C));
  return (size_t)d->B * (size_t)((d->L + S - 1) / S) * (size_t)d->C * sizeof(float);
}

extern "C" gdn2_status gdn2_gated_fwd(const gdn2_gated_desc* d, const void* x, const void* g, const float* h0,
                                      const int32_t* h_index, const int32_t* lengths, const uint8_t* reset, void* h,
                                      float* last, float* marks, uint32_t* flags, void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_gated(d);
  if (s != GDN2_OK) return s;
  if (!last || !flags || (d->L && (!x || !g || !h))) return GDN2_ERR_INVALID_ARGUMENT;
  if (h_index ? !h0 || d->n_states < 1 : h0 && d->n_states != d->B) return GDN2_ERR_INVALID_ARGUMENT;
  const size_t n = access(d);
  if (off(x, n) || off(g, n) || off(h, n) || off(h0, 4) || off(last, 4) || off(marks, 4) || off(flags, 4) ||
      off(lengths, 4) || off(h_index, 4))
    return GDN2_ERR_INVALID_ARGUMENT;
  GatedParams p = params_of(d);
  p.x = x; p.g = g; p.h0 = h0; p.index = h_index; p.lengths = lengths; p.reset = reset;
  p.h = h; p.last = last; p.marks = marks; p.flags = flags;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d->L <= kStepTokens && !marks) {
    const int V = pairs(d) ? 2 : 1;
    const unsigned grid = (unsigned)(((long long)d->B * ((d->C + V - 1) / V) + 127) / 128);
    if (d->dtype == GDN2_F32) gated_step_kernel<float, 1><<<grid, 128, 0, st>>>(p);
    else if (V == 2) gated_step_kernel<__nv_bfloat16, 2><<<grid, 128, 0, st>>>(p);
    else gated_step_kernel<__nv_bfloat16, 1><<<grid, 128, 0, st>>>(p);
    e = cudaGetLastError();
  } else if (d->dtype == GDN2_F32) {
    e = launch_gated<float>(false, p, st);
  } else {
    e = launch_gated<__nv_bfloat16>(false, p, st);
  }
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}

extern "C" gdn2_status gdn2_gated_bwd(const gdn2_gated_desc* d, const void* x, const void* g, const int32_t* lengths,
                                      const uint8_t* reset, const float* marks, const void* dh, const float* dlast,
                                      void* dx, void* dg, float* dh0, uint32_t* flags, void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_gated(d);
  if (s != GDN2_OK) return s;
  if (d->L < 1 || !x || !g || !marks || !dh || !dx || !dg || !flags) return GDN2_ERR_INVALID_ARGUMENT;
  const size_t n = access(d);
  if (off(x, n) || off(g, n) || off(dh, n) || off(dx, n) || off(dg, n) || off(marks, 4) || off(dlast, 4) ||
      off(dh0, 4) || off(lengths, 4) || off(flags, 4))
    return GDN2_ERR_INVALID_ARGUMENT;
  GatedParams p = params_of(d);
  p.x = x; p.g = g; p.lengths = lengths; p.reset = reset; p.marks = const_cast<float*>(marks);
  p.dy = dh; p.dlast = dlast; p.dx = dx; p.dg = dg; p.dh0 = dh0; p.flags = flags;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == GDN2_F32 ? launch_gated<float>(true, p, st)
                                             : launch_gated<__nv_bfloat16>(true, p, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
