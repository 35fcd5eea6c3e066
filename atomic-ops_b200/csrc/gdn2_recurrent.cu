// The recurrent form of the GDN-2 operator (sm_100a): any number of tokens, one at a time.
//
// Per head, with the state S (d_k x d_v, fp32) and per token t
//   a = exp(min(g_t, 0)),  bk = b_t k_t,
//   d = w_t v_t - bk^T (diag(a) S),   S <- diag(a) S + k_t d^T,   o_t = scale q_t^T S.
// It is the token recurrence that the chunked operator evaluates 128 tokens at a time (with
// wy_eps = 0: nothing is damped here).  Columns of S (d_v) are independent of one another, so a
// head's columns are split over CTAs and warps freely; the reductions run over d_k only.  All
// arithmetic and the state are fp32; bf16 inputs are widened as they are loaded.
#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

struct RecParams {
  const void *q, *k, *v, *w, *b, *g;
  long long sb[6], sh[6], sl[6];  // element strides of q, k, v, w, b, g over B, H, L
  long long ob, oh, ol;           // element strides of o
  const float* h0;                // (n_states, H, D, D), or null for zeros
  const int32_t* h_index;         // (B) rows of h0, negative: zeros; null: row b
  const int32_t* lengths;         // (B) valid tokens, or null for L
  float* o;
  float* h_out;                   // (B, H, D, D)
  uint32_t* flags;                // [0] a positive gate was seen, [1] an index or length out of range was seen
  int H, L, n_states;
  float scale, clip;
};

// The state row of sequence b in h0, or -1 for zeros.
__device__ __forceinline__ int state_row(const RecParams& p, int b, bool report) {
  if (!p.h0) return -1;
  if (!p.h_index) return b;
  const int r = __ldg(p.h_index + b);
  if (r >= p.n_states) {
    if (report) p.flags[1] = 1u;
    return -1;
  }
  return r < 0 ? -1 : r;
}
__device__ __forceinline__ int valid_len(const RecParams& p, int b, bool report) {
  if (!p.lengths) return p.L;
  const int n = __ldg(p.lengths + b);
  if (n < 0 || n > p.L) {
    if (report) p.flags[1] = 1u;
    return n < 0 ? 0 : p.L;
  }
  return n;
}

// ---------------------------------------------------------------------------------------------
// One token (or none).  The call moves the states once through the SMs: one CTA holds CW columns
// of a head's state in registers (a thread has four neighbouring columns of CW / 8 rows).  Both
// products read the undecayed state, r = (bk a)^T S and p = (q a)^T S, so one reduction serves
// them: d = w v - r, o = scale (p + (q . k) d).
// ---------------------------------------------------------------------------------------------
constexpr int kStepThreads = 256;

template <class T, int CW>
__global__ void __launch_bounds__(kStepThreads) rec_step_kernel(RecParams p) {
  constexpr int kCols4 = CW / 4;                    // threads along a row
  constexpr int kRowsPass = kStepThreads / kCols4;  // rows per pass
  constexpr int kR = kD / kRowsPass;                // rows per thread
  constexpr int kWarps = kStepThreads / 32;
  __shared__ float4 vec[kD];  // a, k, b k a, q a scale
  __shared__ float wv[CW];
  __shared__ float qk_part[kD / 32];
  __shared__ float4 red[kWarps][2][kCols4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
  const int c0 = blockIdx.y * CW;
  const int cx = tid % kCols4, ry = tid / kCols4;
  const bool first = tid == 0 && h == 0 && blockIdx.y == 0;
  const int row = state_row(p, b, first);
  const int n = valid_len(p, b, first);
  const size_t tile = (size_t)ry * kD + c0 + cx * 4;
  float4 s[kR];
  if (row >= 0) {
    const float* src = p.h0 + ((size_t)row * p.H + h) * (kD * kD) + tile;
#pragma unroll
    for (int i = 0; i < kR; ++i) s[i] = *reinterpret_cast<const float4*>(src + (size_t)i * kRowsPass * kD);
  } else {
#pragma unroll
    for (int i = 0; i < kR; ++i) s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float* dst = p.h_out + (size_t)bh * (kD * kD) + tile;
  if (n == 0) {
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const float4 x = s[i];
      *reinterpret_cast<float4*>(dst + (size_t)i * kRowsPass * kD) =
          make_float4(sanitize(x.x, p.clip), sanitize(x.y, p.clip), sanitize(x.z, p.clip), sanitize(x.w, p.clip));
    }
    if (p.L > 0 && tid < CW) p.o[b * p.ob + h * p.oh + c0 + tid] = 0.f;
    return;
  }
  if (tid < kD) {
    const float q = ld1(static_cast<const T*>(p.q) + b * p.sb[0] + h * p.sh[0] + tid) * p.scale;
    const float k = ld1(static_cast<const T*>(p.k) + b * p.sb[1] + h * p.sh[1] + tid);
    const float be = ld1(static_cast<const T*>(p.b) + b * p.sb[4] + h * p.sh[4] + tid);
    const float g = ld1(static_cast<const T*>(p.g) + b * p.sb[5] + h * p.sh[5] + tid);
    if (g > 0.f) p.flags[0] = 1u;
    const float a = expf(fminf(g, 0.f));
    vec[tid] = make_float4(a, k, be * k * a, q * a);
    float qk = q * k;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, m);
    if (lane == 0) qk_part[warp] = qk;
  } else if (tid - kD < CW) {
    const int c = c0 + tid - kD;
    wv[tid - kD] = ld1(static_cast<const T*>(p.v) + b * p.sb[2] + h * p.sh[2] + c) *
                   ld1(static_cast<const T*>(p.w) + b * p.sb[3] + h * p.sh[3] + c);
  }
  __syncthreads();
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f), o = r;
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const float4 f = vec[ry + i * kRowsPass];
    r.x = fmaf(f.z, s[i].x, r.x); r.y = fmaf(f.z, s[i].y, r.y);
    r.z = fmaf(f.z, s[i].z, r.z); r.w = fmaf(f.z, s[i].w, r.w);
    o.x = fmaf(f.w, s[i].x, o.x); o.y = fmaf(f.w, s[i].y, o.y);
    o.z = fmaf(f.w, s[i].z, o.z); o.w = fmaf(f.w, s[i].w, o.w);
  }
  // threads of a warp that share columns (kCols4 < 32), then the warps
#pragma unroll
  for (int m = 16; m >= kCols4; m >>= 1) {
    r.x += __shfl_xor_sync(0xffffffffu, r.x, m); r.y += __shfl_xor_sync(0xffffffffu, r.y, m);
    r.z += __shfl_xor_sync(0xffffffffu, r.z, m); r.w += __shfl_xor_sync(0xffffffffu, r.w, m);
    o.x += __shfl_xor_sync(0xffffffffu, o.x, m); o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
    o.z += __shfl_xor_sync(0xffffffffu, o.z, m); o.w += __shfl_xor_sync(0xffffffffu, o.w, m);
  }
  if (lane < kCols4) {
    red[warp][0][cx] = r;
    red[warp][1][cx] = o;
  }
  __syncthreads();
  r = make_float4(0.f, 0.f, 0.f, 0.f);
  o = r;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const float4 x = red[i][0][cx], y = red[i][1][cx];
    r.x += x.x; r.y += x.y; r.z += x.z; r.w += x.w;
    o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
  }
  const float4 u = *reinterpret_cast<const float4*>(&wv[cx * 4]);
  const float4 d = make_float4(u.x - r.x, u.y - r.y, u.z - r.z, u.w - r.w);
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const float4 f = vec[ry + i * kRowsPass];
    float4 x = s[i];
    x.x = sanitize(fmaf(f.y, d.x, f.x * x.x), p.clip);
    x.y = sanitize(fmaf(f.y, d.y, f.x * x.y), p.clip);
    x.z = sanitize(fmaf(f.y, d.z, f.x * x.z), p.clip);
    x.w = sanitize(fmaf(f.y, d.w, f.x * x.w), p.clip);
    *reinterpret_cast<float4*>(dst + (size_t)i * kRowsPass * kD) = x;
  }
  if (ry == 0) {
    const float qk = qk_part[0] + qk_part[1] + qk_part[2] + qk_part[3];
    *reinterpret_cast<float4*>(p.o + b * p.ob + h * p.oh + c0 + cx * 4) =
        make_float4(sanitize(fmaf(qk, d.x, o.x), p.clip), sanitize(fmaf(qk, d.y, o.y), p.clip),
                    sanitize(fmaf(qk, d.z, o.z), p.clip), sanitize(fmaf(qk, d.w, o.w), p.clip));
  }
}

// ---------------------------------------------------------------------------------------------
// Several tokens.  A warp owns kM columns per group of eight lanes and keeps them in registers
// over all tokens (16 rows each lane), so the token loop reduces inside the warp and waits for
// no other warp; the tokens' vectors are staged in shared memory for the whole CTA.
// ---------------------------------------------------------------------------------------------
constexpr int kSeqWarps = 4;
constexpr int kSeqTok = 8;  // tokens staged at a time

template <class T, int kM>
__global__ void __launch_bounds__(kSeqWarps * 32) rec_seq_kernel(RecParams p) {
  constexpr int kCols = kSeqWarps * 4 * kM;  // columns of a CTA
  __shared__ float sa[kSeqTok][kD], sk[kSeqTok][kD], sbk[kSeqTok][kD], sq[kSeqTok][kD], swv[kSeqTok][kCols];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
  const int c0 = blockIdx.y * kCols;
  const int rg = lane & 7, cg = lane >> 3;
  const int cw = (warp * 4 + cg) * kM;  // this lane's first column within the CTA
  const bool first = tid == 0 && h == 0 && blockIdx.y == 0;
  const int row = state_row(p, b, first);
  const int n = valid_len(p, b, first);
  // lane rg holds rows 4 rg + 32 i + j (i, j < 4)
  float s[16][kM];
  const size_t at = (size_t)c0 + cw;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = rg * 4 + (i >> 2) * 32 + (i & 3);
#pragma unroll
    for (int m = 0; m < kM; ++m)
      s[i][m] = row >= 0 ? p.h0[((size_t)row * p.H + h) * (kD * kD) + (size_t)r * kD + at + m] : 0.f;
  }
  float* op = p.o + b * p.ob + h * p.oh + c0 + cw;
  for (int t0 = 0; t0 < n; t0 += kSeqTok) {
    const int tc = min(kSeqTok, n - t0);
    __syncthreads();
    for (int i = tid; i < tc * kD; i += kSeqWarps * 32) {
      const int t = i / kD, d = i % kD;
      const long long l = t0 + t;
      const float k = ld1(static_cast<const T*>(p.k) + b * p.sb[1] + h * p.sh[1] + l * p.sl[1] + d);
      const float be = ld1(static_cast<const T*>(p.b) + b * p.sb[4] + h * p.sh[4] + l * p.sl[4] + d);
      const float g = ld1(static_cast<const T*>(p.g) + b * p.sb[5] + h * p.sh[5] + l * p.sl[5] + d);
      if (g > 0.f) p.flags[0] = 1u;
      sq[t][d] = p.scale * ld1(static_cast<const T*>(p.q) + b * p.sb[0] + h * p.sh[0] + l * p.sl[0] + d);
      sk[t][d] = k;
      sbk[t][d] = be * k;
      sa[t][d] = expf(fminf(g, 0.f));
    }
    for (int i = tid; i < tc * kCols; i += kSeqWarps * 32) {
      const int t = i / kCols, c = i % kCols;
      const long long l = t0 + t;
      swv[t][c] = ld1(static_cast<const T*>(p.v) + b * p.sb[2] + h * p.sh[2] + l * p.sl[2] + c0 + c) *
                  ld1(static_cast<const T*>(p.w) + b * p.sb[3] + h * p.sh[3] + l * p.sl[3] + c0 + c);
    }
    __syncthreads();
    for (int t = 0; t < tc; ++t) {
      float r[kM], o[kM];
#pragma unroll
      for (int m = 0; m < kM; ++m) r[m] = o[m] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = *reinterpret_cast<const float4*>(&sa[t][rg * 4 + i * 32]);
        const float4 bk = *reinterpret_cast<const float4*>(&sbk[t][rg * 4 + i * 32]);
        const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {bk.x, bk.y, bk.z, bk.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            s[i * 4 + j][m] *= av[j];
            r[m] = fmaf(bv[j], s[i * 4 + j][m], r[m]);
          }
      }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1)
#pragma unroll
        for (int m = 0; m < kM; ++m) r[m] += __shfl_xor_sync(0xffffffffu, r[m], x);
#pragma unroll
      for (int m = 0; m < kM; ++m) r[m] = swv[t][cw + m] - r[m];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 kk = *reinterpret_cast<const float4*>(&sk[t][rg * 4 + i * 32]);
        const float4 q = *reinterpret_cast<const float4*>(&sq[t][rg * 4 + i * 32]);
        const float kv[4] = {kk.x, kk.y, kk.z, kk.w}, qv[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            s[i * 4 + j][m] = fmaf(kv[j], r[m], s[i * 4 + j][m]);
            o[m] = fmaf(qv[j], s[i * 4 + j][m], o[m]);
          }
      }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1)
#pragma unroll
        for (int m = 0; m < kM; ++m) o[m] += __shfl_xor_sync(0xffffffffu, o[m], x);
      if (rg == 0) {
#pragma unroll
        for (int m = 0; m < kM; ++m) op[(t0 + t) * p.ol + m] = sanitize(o[m], p.clip);
      }
    }
  }
  for (int i = n * kCols + tid; i < p.L * kCols; i += kSeqWarps * 32)  // past the sequence's end
    p.o[b * p.ob + h * p.oh + (i / kCols) * p.ol + c0 + i % kCols] = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = rg * 4 + (i >> 2) * 32 + (i & 3);
#pragma unroll
    for (int m = 0; m < kM; ++m)
      p.h_out[(size_t)bh * (kD * kD) + (size_t)r * kD + at + m] = sanitize(s[i][m], p.clip);
  }
}

template <class T>
void launch(const RecParams& p, int BH, cudaStream_t st) {
  if (p.L <= 1) {
    rec_step_kernel<T, 128><<<dim3(BH, 1), kStepThreads, 0, st>>>(p);
  } else {
    rec_seq_kernel<T, 2><<<dim3(BH, kD / (kSeqWarps * 8)), kSeqWarps * 32, 0, st>>>(p);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace gdn2

extern "C" gdn2_status gdn2_recurrent(const gdn2_rec_desc* d, const void* q, const void* k, const void* v,
                                      const void* w, const void* b, const void* g, const float* h0,
                                      const int32_t* h_index, const int32_t* lengths, float* o, float* h_out,
                                      uint32_t* flags, void* stream) {
  using namespace gdn2;
  if (!d || d->B <= 0 || d->H <= 0 || d->L < 0 || d->D <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->in_dtype != GDN2_F32 && d->in_dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (!(d->clip > 0.f) || (int64_t)d->B * d->H > 0x7fffffffLL) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->D != kD) return GDN2_ERR_UNSUPPORTED;
  const int el = d->in_dtype == GDN2_BF16 ? 2 : 4;
  const void* ins[6] = {q, k, v, w, b, g};
  RecParams p{};
  if (d->L > 0) {
    for (int i = 0; i < 6; ++i) {
      if (!ins[i] || !aligned16(ins[i])) return GDN2_ERR_INVALID_ARGUMENT;
      for (int j = 0; j < 3; ++j)
        if (d->stride[i][j] < 0 || (d->stride[i][j] * el) % 16) return GDN2_ERR_INVALID_ARGUMENT;
    }
    if (!o || !aligned16(o)) return GDN2_ERR_INVALID_ARGUMENT;
    for (int j = 0; j < 3; ++j)
      if (d->o_stride[j] < 0 || d->o_stride[j] % 4) return GDN2_ERR_INVALID_ARGUMENT;
  }
  if (!h_out || !aligned16(h_out) || !flags || (h0 && !aligned16(h0))) return GDN2_ERR_INVALID_ARGUMENT;
  if (h0 && (d->n_states <= 0 || (!h_index && d->n_states < d->B))) return GDN2_ERR_INVALID_ARGUMENT;
  if (h0 == h_out && h_index) return GDN2_ERR_INVALID_ARGUMENT;  // another sequence may still read the row
  p.q = q; p.k = k; p.v = v; p.w = w; p.b = b; p.g = g;
  for (int i = 0; i < 6; ++i) {
    p.sb[i] = d->stride[i][0];
    p.sh[i] = d->stride[i][1];
    p.sl[i] = d->stride[i][2];
  }
  p.ob = d->o_stride[0]; p.oh = d->o_stride[1]; p.ol = d->o_stride[2];
  p.h0 = h0; p.h_index = h_index; p.lengths = lengths; p.o = o; p.h_out = h_out; p.flags = flags;
  p.H = d->H; p.L = d->L; p.n_states = d->n_states;
  p.scale = d->scale; p.clip = d->clip;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (el == 2) launch<__nv_bfloat16>(p, d->B * d->H, st);
  else launch<float>(p, d->B * d->H, st);
  return cudaGetLastError() == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
