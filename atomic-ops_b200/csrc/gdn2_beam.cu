// One step of beam search (sm_100a): from a vocabulary's logits for B x K beams and the beams'
// running scores, the K best continuations of each of the B sequences.
//   logp = (x - m) - log sum exp(x - m),  m = max x,   total = score + logp
// Order: inside a beam by logit, the lowest token first among equals; over a sequence's beams by
// total, the lowest beam first among equals.  A NaN logit or score counts as -inf, a +inf logit as
// the largest finite value; a beam whose logits are all -inf offers totals of -inf.  A finished
// beam offers itself alone: (eos, its score).
//
// The logits are read once.  A warp keeps the R = min(K, V) best of what it has seen as a sorted
// list over its lanes (R <= 32), together with the running maximum and sum of the softmax; most
// values are below the list's last, which one comparison and a vote find out.  Keys join the
// order-preserving bits of the logit with the inverted index, so that no two are equal and the
// result does not depend on the order of insertion.
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
__device__ __forceinline__ float clean(float x) {
  return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}

// Inserts each lane's key (0: none) that is above the list's R-th into the warp's sorted list.
__device__ __forceinline__ void insert(u64& list, u64 key, int R, int lane) {
  u64 last = __shfl_sync(kFull, list, R - 1);
  unsigned todo = __ballot_sync(kFull, key > last);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const u64 k = __shfl_sync(kFull, key, src);
    const unsigned above = __ballot_sync(kFull, list > k);  // a prefix of the lanes
    const u64 up = __shfl_up_sync(kFull, list, 1);
    const int pos = __popc(above);
    if (lane == pos) list = k;
    else if (lane > pos) list = up;
    last = __shfl_sync(kFull, list, R - 1);
    todo &= __ballot_sync(kFull, key > last);
  }
}

// max and sum of exp(x - max) of two parts
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, 0.f);
  return make_float2(m, a.y * expf(a.x - m) + b.y * expf(b.x - m));
}

constexpr int kScanWarps = 8;

// One row's slice: list and softmax statistics into the workspace.
template <class T>
__global__ void __launch_bounds__(kScanWarps * 32) beam_scan_kernel(BeamParams p) {
  __shared__ u64 lists[kScanWarps][32];
  __shared__ float2 stats[kScanWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, split = blockIdx.y;
  if (p.finished && p.finished[row]) return;
  const T* x = static_cast<const T*>(p.logits) + (row / p.K) * p.sb + (row % p.K) * p.sk;
  const int v0 = split * p.slice, v1 = min(p.V, v0 + p.slice);
  u64 list = 0;
  float2 st = make_float2(-INFINITY, 0.f);
  for (int v = v0 + warp * 32; v < v1; v += kScanWarps * 32) {
    const int i = v + lane;
    u64 key = 0;
    if (i < v1) {
      const float f = clean(ld1(x + i));
      key = make_key(f, i);
      if (f > st.x) {
        st.y = st.y * expf(st.x - f) + 1.f;
        st.x = f;
      } else if (f > -INFINITY) {
        st.y += expf(f - st.x);
      }
    }
    insert(list, key, p.R, lane);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
    st = join(st, make_float2(__shfl_xor_sync(kFull, st.x, m), __shfl_xor_sync(kFull, st.y, m)));
  lists[warp][lane] = lane < p.R ? list : 0;
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  if (warp) return;
#pragma unroll 1
  for (int i = 1; i < kScanWarps; ++i) {
    insert(list, lists[i][lane], p.R, lane);
    st = join(st, stats[i]);
  }
  const size_t at = (size_t)row * p.splits + split;
  if (lane < p.R) p.lists[at * p.R + lane] = list;
  if (lane == 0) p.stats[at] = st;
}

// One sequence: joins its beams' slices (a warp per beam) and selects over them.
__global__ void __launch_bounds__(1024) beam_pick_kernel(BeamParams p) {
  __shared__ float total[32 * 32];
  __shared__ int token[32 * 32];
  const int tid = threadIdx.x, lane = tid & 31, k = tid >> 5;
  const int b = blockIdx.x, row = b * p.K + k;
  const float score0 = p.scores[row];
  const float score = score0 != score0 ? -INFINITY : score0;
  if (p.finished && p.finished[row]) {
    total[k * 32 + lane] = lane == 0 ? score : -INFINITY;
    token[k * 32 + lane] = p.eos;
  } else {
    u64 list = 0;
    float2 st = make_float2(-INFINITY, 0.f);
    for (int s = 0; s < p.splits; ++s) {
      const size_t at = (size_t)row * p.splits + s;
      insert(list, lane < p.R ? p.lists[at * p.R + lane] : 0, p.R, lane);
      st = join(st, p.stats[at]);
    }
    float t = -INFINITY;
    if (lane < p.R && st.x > -INFINITY) {
      t = score + ((key_value(list) - st.x) - logf(st.y));
      if (t != t) t = -INFINITY;
    }
    total[k * 32 + lane] = t;
    token[k * 32 + lane] = (int)key_index(list);
  }
  __syncthreads();
  if (k) return;
  u64 best = 0;
  for (int j = 0; j < p.K; ++j)  // a beam's totals fall with the rank: ranks past R never matter
    insert(best, lane < p.R ? make_key(total[j * 32 + lane], j * 32 + lane) : 0, p.K, lane);
  if (lane < p.K) {
    const int c = (int)key_index(best), tok = token[c], parent = b * p.K + c / 32;
    const int at = b * p.K + lane;
    p.out_scores[at] = total[c];
    p.out_row[at] = parent;
    p.out_token[at] = tok;
    p.out_finished[at] = (p.finished && p.finished[parent]) || tok == p.eos;
  }
}

struct BeamPlan { int R, splits, slice; size_t stats, total; };
BeamPlan beam_plan(const gdn2_beam_desc* d) {
  BeamPlan pl{};
  pl.R = d->K < d->V ? d->K : d->V;
  const long long rows = (long long)d->B * d->K;
  // enough slices to cover the GPU a few times over, none smaller than 4096 values
  long long want = rows >= 592 ? 1 : 592 / rows, most = (d->V + 4095) / 4096;
  pl.splits = (int)(want < most ? want : most);
  pl.slice = (d->V + pl.splits - 1) / pl.splits;
  pl.stats = ((size_t)rows * pl.splits * pl.R * 8 + 255) / 256 * 256;
  pl.total = pl.stats + (size_t)rows * pl.splits * 8;
  return pl;
}
gdn2_status check_beam(const gdn2_beam_desc* d) {
  if (!d || d->B <= 0 || d->K <= 0 || d->V <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->stride_b < 0 || d->stride_k < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->K > 32 || (int64_t)d->B * d->K > (1 << 30)) return GDN2_ERR_UNSUPPORTED;
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
  if (!logits || !scores || !out_scores || !out_row || !out_token || !out_finished || !workspace ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return GDN2_ERR_INVALID_ARGUMENT;
  const BeamPlan pl = beam_plan(d);
  BeamParams p{};
  p.logits = logits; p.sb = d->stride_b; p.sk = d->stride_k;
  p.scores = scores; p.finished = finished;
  p.out_scores = out_scores; p.out_row = out_row; p.out_token = out_token; p.out_finished = out_finished;
  p.lists = static_cast<u64*>(workspace);
  p.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + pl.stats);
  p.B = d->B; p.K = d->K; p.V = d->V; p.R = pl.R; p.splits = pl.splits; p.slice = pl.slice; p.eos = d->eos;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(d->B * d->K, pl.splits);
  if (d->dtype == GDN2_BF16) beam_scan_kernel<__nv_bfloat16><<<grid, kScanWarps * 32, 0, st>>>(p);
  else beam_scan_kernel<float><<<grid, kScanWarps * 32, 0, st>>>(p);
  beam_pick_kernel<<<d->B, d->K * 32, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
