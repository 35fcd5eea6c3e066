// One step of beam search (sm_100a): from a vocabulary's logits for B x K beams and the beams'
// running scores, the K best continuations of each of the B sequences.
//   logp = (x - m) - log sum exp(x - m),  m = max x,   total = score + logp
// Order: inside a beam by logit, the lowest token first among equals; over a sequence's beams by
// total, the lowest beam first among equals.  A NaN logit or score counts as -inf, a +inf logit as
// the largest finite value; a beam whose logits are all -inf offers totals of -inf.  A finished
// beam offers itself alone: (eos, its score).
//
// The logits are read once (a few lanes' of them twice), and the waits for them bound the call where there are
// many; the exponentials (a quarter of an SM's lanes a cycle) come next.  A warp takes 256 values at a time,
// eight to a lane, and a lane keeps the running maximum and sum of its values' softmax.  With R = min(K, V) <= 32,
// R lanes' maxima bound the R best values from below; only the few lanes whose maximum reaches the bound are
// looked through again, value by value, into a sorted list over the warp's lanes.  Keys join the order-preserving
// bits of the logit with the inverted index, so that no two are equal and the result does not depend on the order
// of insertion.
//
// Small vocabularies take one launch (a CTA per sequence); else a first launch reads the logits, a
// long row's slices spread over CTAs, and a second one, started while the first still runs, joins them.
#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

using u64 = unsigned long long;
constexpr unsigned kFull = 0xffffffffu;

struct BeamParams {
  const void* logits;
  long long sb, sk;       // element strides over B and K (V contiguous)
  const float* scores;    // (B, K)
  const uint8_t* finished;  // (B, K) or null
  float* out_scores;      // (B, K)
  int32_t* out_row;
  int32_t* out_token;
  uint8_t* out_finished;
  u64* lists;             // workspace: (B K, splits, R) keys
  float2* stats;          // workspace: (B K, splits) max and sum
  int B, K, V, R, splits, slice, eos;
};

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 make_key(float x, uint32_t index) {
  return ((u64)ordered(x + 0.f) << 32) | (uint32_t)~index;  // + 0: -0 and 0 are equal
}
__device__ __forceinline__ float key_value(u64 k) { return from_ordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }
__device__ __forceinline__ float clean(float x) {  // NaN: -inf; +inf: the largest finite value
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);
}

// Sorts 32 keys over the lanes, largest first (bitonic).  Like insert() a function of its own: inlined
// wherever they are used they are most of the kernels' code, and fetching that costs more than calls do.
__device__ __noinline__ u64 sort32(u64 k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int m = size >> 1; m > 0; m >>= 1) {
      const u64 other = __shfl_xor_sync(kFull, k, m);
      const bool down = (lane & size) == 0, low = (lane & m) == 0;
      k = (down == low) == (k > other) ? k : other;
    }
  return k;
}

// The warp's sorted list with each lane's key (0: none) that is above its R-th inserted.
__device__ __noinline__ u64 inserted(u64 list, u64 key, int R, int lane) {
  u64 last = __shfl_sync(kFull, list, R - 1);
  unsigned todo = __ballot_sync(kFull, key > last);
  if (__popc(todo) > 6) {  // sort them and take the upper half of the two lists' merge
    const u64 k = sort32(key, lane);
    const u64 back = __shfl_sync(kFull, k, 31 - lane);
    u64 m = list > back ? list : back;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const u64 other = __shfl_xor_sync(kFull, m, d);
      m = ((lane & d) == 0) == (m > other) ? m : other;
    }
    return m;
  }
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const u64 k = __shfl_sync(kFull, key, src);
    const unsigned above = __ballot_sync(kFull, list > k);  // a prefix of the lanes
    const u64 up = __shfl_up_sync(kFull, list, 1);
    const int pos = __popc(above);
    if (lane == pos) list = k;
    else if (lane > pos) list = up;
  }
  return list;
}
__device__ __forceinline__ void insert(u64& list, u64 key, int R, int lane) { list = inserted(list, key, R, lane); }
// The best of n keys in memory (0: none), into the warp's list.
__device__ __forceinline__ void gather(u64& list, const u64* keys, int n, int R, int lane) {
  for (int i = 0; i < n; i += 128) {
    u64 k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = i + j * 32 + lane < n ? keys[i + j * 32 + lane] : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * 32 < n) insert(list, k[j], R, lane);
  }
}

// max and sum of exp(x - max) of two parts
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, 0.f);
  return make_float2(m, a.y * expf(a.x - m) + b.y * expf(b.x - m));
}
__device__ __forceinline__ float2 join_warp(float2 st) {
  float m = st.x;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, i));
  float s = m > -INFINITY ? st.y * expf(st.x - m) : 0.f;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(kFull, s, i);
  return make_float2(m, s);
}
// e^x for x <= 0: rounding x log2 e costs at most |x| 2^-23 of the value, the instruction 2^-22.  Over a row's sum
// that is at most ln V 2^-23 + 2^-22 (|x| has a mean of ln V or less under the softmax), and as much in its logarithm.
__device__ __forceinline__ float exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// The lane's share of x[v0, v1): the warp takes pieces of 256 values, `first` of `stride`, and a lane
// every 32nd of a piece.  That needs no alignment of the rows, and which values are summed in which
// order depends on their place in the row alone.  scan() returns the lane's maximum and sum; the
// maximum is also the lane's best candidate.
struct Pieces {
  int at, hop, count;  // this lane's first value, distance between its pieces, pieces of the warp
};
__device__ __forceinline__ Pieces pieces(int v0, int v1, int first, int stride, int lane) {
  const int start = v0 + first * 256;
  return {start + lane, stride * 256, start < v1 ? (v1 - start + stride * 256 - 1) / (stride * 256) : 0};
}
__device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(__ldg(p)); }
__device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) {
  return (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16;
}
template <class T>
__device__ __forceinline__ float2 scan(const T* x, int v1, const Pieces& pc) {
  float m = -INFINITY, sum = 0.f;
  float next[8];  // a piece is on its way while one is worked on (two or four: no faster, more code to fetch)
  auto fetch = [&](int i) {
    const int from = pc.at + i * pc.hop;
    const T* src = x + from;
    if (i < pc.count && from + 7 * 32 < v1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) next[j] = __uint_as_float(bits(src + j * 32));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) next[j] = i < pc.count && from + j * 32 < v1 ? __uint_as_float(bits(src + j * 32)) : -INFINITY;
    }
  };
  fetch(0);
  for (int i = 0; i < pc.count; ++i) {
    float c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = next[j];
    fetch(i + 1);
    for (int again = 0; again < 2; ++again) {
      float top = c[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, c[j]);
      const float big = fmaxf(m, top);
      float part = sum;
      if (big > m) part *= exp_fast(m - big);
      if (big > -INFINITY) {
#pragma unroll
        for (int j = 0; j < 8; ++j) part += exp_fast(c[j] - big);
      }
      if (part == part) {
        m = big;
        sum = part;
        break;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = clean(c[j]);  // a NaN or +inf among the values
    }
  }
  return make_float2(m, sum);
}
// The q-th largest of the lanes' values.
__device__ __forceinline__ float nth(float v, int q, int lane) {
  if (q > 4) return key_value(__shfl_sync(kFull, sort32(make_key(v, lane), lane), q - 1));
  float r = v;
  for (int i = 0; i < q; ++i) {
    r = v;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) r = fmaxf(r, __shfl_xor_sync(kFull, r, m));
    const unsigned who = __ballot_sync(kFull, v == r);
    if (lane == __ffs(who) - 1) v = -INFINITY;
  }
  return r;
}
// Four candidates a lane, x[at] where at < v1, into the warp's list.
template <class T>
__device__ __forceinline__ void offer(u64& list, const T* x, int v1, const int at[4], float least, int R, int lane) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = at[i] < v1 ? bits(x + at[i]) : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = clean(__uint_as_float(u[i]));
    const bool on = at[i] < v1 && v >= least;
    if (__any_sync(kFull, on)) insert(list, on ? make_key(v, at[i]) : 0, R, lane);
  }
}
// The warp's candidates into its list: the values, `least` or more, of the lanes whose maximum is that.
// Those lanes' values are read again by the whole warp: one lane's after the other's, or, where a lane has
// fewer than 32, several lanes' at a time.
template <class T>
__device__ __forceinline__ void collect(u64& list, const T* x, int v1, const Pieces& pc, float m, float least, int R,
                                        int lane, uint8_t lanes[32]) {
  unsigned who = __ballot_sync(kFull, m >= least);
  const int own = pc.at - lane, each = pc.count * 8;
  int at[4];
  if (each >= 32) {
    while (who) {
      const int from = own + __ffs(who) - 1;
      who &= who - 1;
      for (int c = lane; c < each + lane; c += 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = c + i * 32;
          at[i] = n < each ? from + (n >> 3) * pc.hop + (n & 7) * 32 : v1;
        }
        offer(list, x, v1, at, least, R, lane);
      }
    }
  } else {
    if (m >= least) lanes[__popc(who & ((1u << lane) - 1))] = (uint8_t)lane;
    __syncwarp();
    const int total = __popc(who) * each;
    for (int c = lane; c < total + lane; c += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = c + i * 32;
        at[i] = n < total ? own + lanes[n / each] + (n % each >> 3) * pc.hop + (n & 7) * 32 : v1;
      }
      offer(list, x, v1, at, least, R, lane);
    }
  }
}

constexpr int kScanWarps = 8;

// One row's slice: list and softmax statistics into the workspace.  Measured (with the joining launch): 32 x 8 x
// 50001 bf16 22.5 us (1.1 TB/s; it issues in 41 % of the cycles and mostly waits for its loads, two bytes a lane
// and one piece ahead; then the lists' latency), 1 x 5 x 262144 fp32 13 us (latency).
template <class T>
__global__ void __launch_bounds__(kScanWarps * 32) beam_scan_kernel(BeamParams p) {
  __shared__ u64 lists[kScanWarps * 32];
  __shared__ float2 stats[kScanWarps];
  __shared__ float bound[kScanWarps];
  __shared__ uint8_t lanes[kScanWarps][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, split = blockIdx.y;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (p.finished && p.finished[row]) return;
  const T* x = static_cast<const T*>(p.logits) + (row / p.K) * p.sb + (row % p.K) * p.sk;
  const int v0 = split * p.slice, v1 = min(p.V, v0 + p.slice);
  const Pieces pc = pieces(v0, v1, warp, kScanWarps, lane);
  float2 st = scan(x, v1, pc);
  // R lanes' maxima are at or above the least of the warps' q-th largest, so the slice's R best are too
  const float top = st.x, mine = nth(top, (p.R + kScanWarps - 1) / kScanWarps, lane);
  if (lane == 0) bound[warp] = mine;
  st = join_warp(st);
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  float least = bound[0];
#pragma unroll
  for (int i = 1; i < kScanWarps; ++i) least = fminf(least, bound[i]);
  u64 list = 0;
  collect(list, x, v1, pc, top, least, p.R, lane, lanes[warp]);
  if (lane < p.R) lists[warp * p.R + lane] = list;
  __syncthreads();
  if (warp) return;
  list = 0;
  gather(list, lists, kScanWarps * p.R, p.R, lane);
  st = join_warp(lane < kScanWarps ? stats[lane] : make_float2(-INFINITY, 0.f));
  const size_t at = (size_t)row * p.splits + split;
  if (lane < p.R) p.lists[at * p.R + lane] = list;
  if (lane == 0) p.stats[at] = st;
}

// Measured as the only launch: 8 x 4 x 256 4.5 us, 64 x 16 x 256 10.7 us: the latency of a few hundred dependent
// steps.
//
// One sequence: joins its beams' parts, `per` warps to a beam, and selects over them.  kWhole: reads
// the logits itself.
template <class T, bool kWhole>
__global__ void __launch_bounds__(1024) beam_pick_kernel(BeamParams p, int per) {
  __shared__ u64 lists[32 * 32];
  __shared__ float2 stats[32];
  __shared__ float total[32 * 32];
  __shared__ int token[32 * 32];
  __shared__ uint8_t lanes[32][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int k = warp / per, part = warp % per, row = blockIdx.x * p.K + k;
  const bool done = p.finished && p.finished[row];
  const float score0 = p.scores[row], score = score0 != score0 ? -INFINITY : score0;
  if constexpr (!kWhole) asm volatile("griddepcontrol.wait;" ::: "memory");
  u64 list = 0;
  float2 st = make_float2(-INFINITY, 0.f);
  if (!done) {
    if constexpr (kWhole) {
      const T* x = static_cast<const T*>(p.logits) + blockIdx.x * p.sb + k * p.sk;
      const Pieces pc = pieces(0, p.V, part, per, lane);
      st = scan(x, p.V, pc);
      // see beam_scan_kernel; here each warp goes by its own lanes
      collect(list, x, p.V, pc, st.x, nth(st.x, p.R, lane), p.R, lane, lanes[warp]);
    } else {
      const int n = (p.splits + per - 1) / per, s0 = part * n, s1 = min(p.splits, s0 + n);
      const size_t at = (size_t)row * p.splits;
      for (int s = s0 + lane; s < s1; s += 32) st = join(st, p.stats[at + s]);
      if (s0 < s1) gather(list, p.lists + (at + s0) * p.R, (s1 - s0) * p.R, p.R, lane);
    }
    st = join_warp(st);
  }
  if (per > 1) {
    if (lane < p.R) lists[warp * p.R + lane] = list;
    if (lane == 0) stats[warp] = st;
    __syncthreads();
    if (part == 0) {
      list = 0;
      gather(list, lists + warp * p.R, per * p.R, p.R, lane);
      st = join_warp(lane < per ? stats[warp + lane] : make_float2(-INFINITY, 0.f));
    }
  }
  if (part == 0) {
    float t = -INFINITY;
    if (done) {
      t = lane == 0 ? score : t;
    } else if (lane < p.R && st.x > -INFINITY) {
      t = score + ((key_value(list) - st.x) - logf(st.y));
      if (t != t) t = -INFINITY;
    }
    total[k * 32 + lane] = t;
    token[k * 32 + lane] = done ? p.eos : (int)key_index(list);
  }
  __syncthreads();
  if (warp) return;
  u64 best = lane < p.R ? make_key(total[lane], lane) : 0;  // a beam's totals fall with the rank
  for (int j = 1; j < p.K; ++j) insert(best, lane < p.R ? make_key(total[j * 32 + lane], j * 32 + lane) : 0, p.K, lane);
  if (lane < p.K) {
    const int c = (int)key_index(best), tok = token[c], parent = blockIdx.x * p.K + c / 32;
    const int at = blockIdx.x * p.K + lane;
    p.out_scores[at] = total[c];
    p.out_row[at] = parent;
    p.out_token[at] = tok;
    p.out_finished[at] = (p.finished && p.finished[parent]) || tok == p.eos;
  }
}

// One launch reads and selects where a sequence's logits are few for its CTA.  Measured (one launch / two,
// us): 8 x 4 x 256 5 / 17, 64 x 8 x 2000 12 / 19, 1 x 5 x 4096 9.5 / 11, 2 x 4 x 8192 10.5 / 10.8,
// 16 x 16 x 4096 28 / 21, 64 x 16 x 8192 46 / 32.
bool whole(const gdn2_beam_desc* d) { return d->V <= 8192 && (long long)d->V * d->K <= 32768; }

struct BeamPlan { int R, splits, slice; size_t stats, total; };
BeamPlan beam_plan(const gdn2_beam_desc* d) {
  BeamPlan pl{};
  pl.R = d->K < d->V ? d->K : d->V;
  if (whole(d)) return pl;
  const long long rows = (long long)d->B * d->K;
  // enough slices to cover the GPU a few times over, none smaller than 4096 values (twice and four times as
  // many: 32 x 8 x 50001 27 -> 31 and 41 us, 1 x 5 x 262144 16 -> 18 us)
  long long want = rows >= 592 ? 1 : 592 / rows, most = (d->V + 4095) / 4096;
  pl.splits = (int)(want < most ? want : most);
  pl.slice = (d->V + pl.splits - 1) / pl.splits;
  pl.stats = ((size_t)rows * pl.splits * pl.R * 8 + 255) / 256 * 256;
  pl.total = pl.stats + (size_t)rows * pl.splits * 8;
  return pl;
}
template <class T>
cudaError_t launch(const BeamParams& p, cudaStream_t st) {
  int per = 32 / p.K;  // warps to a beam
  if (p.splits == 0) {
    const int most = p.V / 512;  // values of a warp, where there are warps enough
    if (per > most) per = most > 1 ? most : 1;
    beam_pick_kernel<T, true><<<p.B, p.K * per * 32, 0, st>>>(p, per);
    return cudaGetLastError();
  }
  beam_scan_kernel<T><<<dim3(p.B * p.K, p.splits), kScanWarps * 32, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int most = (p.splits * p.R + 31) / 32;
  if (per > most) per = most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.B);
  cfg.blockDim = dim3(p.K * per * 32);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_pick_kernel<T, false>, p, per);
}
gdn2_status check_beam(const gdn2_beam_desc* d) {
  if (!d || d->B <= 0 || d->K <= 0 || d->V <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->stride_b < 0 || d->stride_k < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->K > 32 || d->V > (1 << 30) || (int64_t)d->B * d->K > (1 << 30)) return GDN2_ERR_UNSUPPORTED;
  return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_beam_workspace_bytes(const gdn2_beam_desc* d) {
  return gdn2::check_beam(d) == GDN2_OK ? gdn2::beam_plan(d).total : 0;
}

extern "C" gdn2_status gdn2_beam_select(const gdn2_beam_desc* d, const void* logits, const float* scores,
                                        const uint8_t* finished, float* out_scores, int32_t* out_row,
                                        int32_t* out_token, uint8_t* out_finished, void* workspace, void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_beam(d);
  if (s != GDN2_OK) return s;
  if (!logits || !scores || !out_scores || !out_row || !out_token || !out_finished) return GDN2_ERR_INVALID_ARGUMENT;
  const BeamPlan pl = beam_plan(d);
  if (pl.total && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))) return GDN2_ERR_INVALID_ARGUMENT;
  const size_t el = d->dtype == GDN2_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(logits) % el) return GDN2_ERR_INVALID_ARGUMENT;
  BeamParams p{};
  p.logits = logits; p.sb = d->stride_b; p.sk = d->stride_k;
  p.scores = scores; p.finished = finished;
  p.out_scores = out_scores; p.out_row = out_row; p.out_token = out_token; p.out_finished = out_finished;
  p.lists = static_cast<u64*>(workspace);
  p.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + pl.stats);
  p.B = d->B; p.K = d->K; p.V = d->V; p.R = pl.R; p.splits = pl.splits; p.slice = pl.slice; p.eos = d->eos;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = el == 2 ? launch<__nv_bfloat16>(p, st) : launch<float>(p, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
