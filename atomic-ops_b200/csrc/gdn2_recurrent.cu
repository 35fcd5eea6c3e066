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

using u64 = unsigned long long;

struct RecParams {
  const void *q, *k, *v, *w, *b, *g;
  long long sb[6], sh[6], sl[6];  // element strides of q, k, v, w, b, g over B, H, L
  long long ob, oh, ol;           // element strides of o
  const float* h0;                // (n_states, H, D, D), or null for zeros
  const int32_t* h_index;         // (B) rows of h0, negative: zeros; null: row b
  const int32_t* lengths;         // (B) valid tokens, or null for L
  float* o;
  float* h_out;                   // (B, H, D, D)
  uint32_t* flags;                // [0] a positive gate was seen, [1] an index or length out of range, [2] a wait ran out
  int H, L, n_states;
  float scale, clip;
  int bf16;                       // the type of q..g, for code that is not compiled for one
};
// 0, or NaN if x is not finite; summed up it tells whether any value was not.
__device__ __forceinline__ float not_finite(float x) { return x * 0.f; }

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
// One token (or none).  The call moves the states once through the SMs: one CTA holds a head's
// state in registers (a thread has four neighbouring columns of 16 rows, a warp whole rows).  Both
// products read the undecayed state, r = (bk a)^T S and p = (q a)^T S, so one reduction serves
// them: d = w v - r, o = scale (p + (q . k) d).  Bound by HBM, 128 KB a head: a CTA's 64 KB of loads are
// in flight before anything is computed.  Measured: 6144 heads 122 us (6.77 TB/s, as fast as a copy), 1536
// heads through an index 32.4 us (6.3 TB/s), 6 heads 3.3 us (a launch).
// ---------------------------------------------------------------------------------------------
constexpr int kStepThreads = 256;

template <class T>
__global__ void __launch_bounds__(kStepThreads) rec_step_kernel(RecParams p) {
  constexpr int kCols4 = kD / 4;                    // threads along a row: a warp
  constexpr int kRowsPass = kStepThreads / kCols4;  // rows per pass
  constexpr int kR = kD / kRowsPass;                // rows per thread
  constexpr int kWarps = kStepThreads / 32;
  __shared__ float4 vec[kD];  // a, k, b k a, q a scale
  __shared__ float wv[kD];
  __shared__ float qk_part[kD / 32];
  __shared__ float4 red[kWarps][2][kCols4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
  const int cx = tid % kCols4, ry = tid / kCols4;
  const bool first = tid == 0 && h == 0;
  const int row = state_row(p, b, first);
  const int n = valid_len(p, b, first);
  const size_t tile = (size_t)ry * kD + cx * 4;
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
    if (p.L > 0 && tid < kD) p.o[b * p.ob + h * p.oh + tid] = 0.f;
    return;
  }
  if (tid < kD) {
    const float q = ld1(static_cast<const T*>(p.q) + b * p.sb[0] + h * p.sh[0] + tid) * p.scale;
    const float k = ld1(static_cast<const T*>(p.k) + b * p.sb[1] + h * p.sh[1] + tid);
    const float be = ld1(static_cast<const T*>(p.b) + b * p.sb[4] + h * p.sh[4] + tid);
    const float g = ld1(static_cast<const T*>(p.g) + b * p.sb[5] + h * p.sh[5] + tid);
    if (g > 0.f) p.flags[0] = 1u;
    const float a = expf(g > 0.f ? 0.f : g);  // a NaN stays one
    vec[tid] = make_float4(a, k, be * k * a, q * a);
    float qk = q * k;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, m);
    if (lane == 0) qk_part[warp] = qk;
  } else {
    const int c = tid - kD;
    wv[c] = ld1(static_cast<const T*>(p.v) + b * p.sb[2] + h * p.sh[2] + c) *
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
  red[warp][0][cx] = r;
  red[warp][1][cx] = o;
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
  const float qk = qk_part[0] + qk_part[1] + qk_part[2] + qk_part[3];
  o = make_float4(fmaf(qk, d.x, o.x), fmaf(qk, d.y, o.y), fmaf(qk, d.z, o.z), fmaf(qk, d.w, o.w));
  // With an infinity about, p + (q . k) d is not q^T S (k_j d and S_j may cancel to a NaN): o is summed from the
  // new state then.  Every warp has all columns, so the warps of the CTA agree.
  const float probe = not_finite(o.x) + not_finite(o.y) + not_finite(o.z) + not_finite(o.w);
  if (__any_sync(0xffffffffu, probe != 0.f)) {
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const float4 f = vec[ry + i * kRowsPass];
      const float q = ld1(static_cast<const T*>(p.q) + b * p.sb[0] + h * p.sh[0] + ry + i * kRowsPass);
      o.x = fmaf(q, fmaf(f.y, d.x, f.x * s[i].x), o.x);
      o.y = fmaf(q, fmaf(f.y, d.y, f.x * s[i].y), o.y);
      o.z = fmaf(q, fmaf(f.y, d.z, f.x * s[i].z), o.z);
      o.w = fmaf(q, fmaf(f.y, d.w, f.x * s[i].w), o.w);
    }
    __syncthreads();  // red is read no more
    red[warp][0][cx] = o;
    __syncthreads();
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < kWarps; ++i) {
      const float4 x = red[i][0][cx];
      o.x = fmaf(p.scale, x.x, o.x); o.y = fmaf(p.scale, x.y, o.y);
      o.z = fmaf(p.scale, x.z, o.z); o.w = fmaf(p.scale, x.w, o.w);
    }
  }
  if (ry == 0)
    *reinterpret_cast<float4*>(p.o + b * p.ob + h * p.oh + cx * 4) =
        make_float4(sanitize(o.x, p.clip), sanitize(o.y, p.clip), sanitize(o.z, p.clip), sanitize(o.w, p.clip));
}

// ---------------------------------------------------------------------------------------------
// Several tokens: blocks of 8.  With G_t the gates summed from the block's start through token t,
//   d_t = w_t v_t - (bk_t e^{G_t})^T S - sum_{s<t} L_ts d_s,
//   o_t = (scale q_t e^{G_t})^T S + sum_{s<=t} P_ts d_s,
//   S  <- diag(e^{G_8}) S + sum_t (k_t e^{G_8 - G_t}) d_t^T,
//   L_ts = sum_d bk_t k_s e^{G_t - G_s},   P_ts = scale sum_d q_t k_s e^{G_t - G_s}
// is the recurrence with the state read once and written once per block: one reduction over d_k
// serves eight tokens, and 3 1/8 products per state element and token are left of 4.  Every factor
// is a product of gates e^g <= 1, so nothing can overflow however far the gates close.
//
// rec_prep_kernel writes what does not depend on S, a record per head and block; rec_wide_kernel or
// rec_deep_kernel walks the records with the state in registers.  X = (I + L)^-1 does not depend on S
// either: the record holds B = X (bk e^G) and V = X (w v), and d = V - B S needs no substitution.
//
// The state's products run on the warp-level tensor instruction (m16n8k8, tf32) with each fp32
// operand split in two (hi lo: 22 bits) and three products; the lo lo product is left out.  That is
// 2^-21 of a product or less, four times fp32's own rounding: errors come out 15 to 20 % above those of a
// plain fp32 form, whose sums they share.  A warp holds the transposed state, 16 columns (d_v)
// x its share of d, in the accumulator layout; the same registers are the next product's first
// operand, since the sum over d may run in any order.  On the CUDA cores the same work is bound by
// the shared-memory traffic of the vectors (every lane needs its own copy), measured 2 to 6 times
// slower.  Sums of the state itself stay outside the tensor instruction, whose additions may
// truncate: U = sum_t k_t d_t^T there, S <- e S + U in fp32.
//
// A value that is not finite reaches every token of its block in these products, and an infinity has no lo.
// It always shows in a d or an o: a CTA that has met one does its columns again from the launch's first
// token on, by the definition, token by token (seq_literal).
// ---------------------------------------------------------------------------------------------
constexpr int kSmCount = 148;  // of a B200
constexpr int kTok = 8;
// A record, in floats, in the order in which the lanes (g = lane / 4, t = lane % 4) read it:
constexpr int kRecDot = 0;               // [16 tiles of d][32 lanes]{B(8j+2t), B(8j+2t+1), q.., q..} of token g
constexpr int kRecK = 16 * 128;          // [8 pairs of tiles][32]{k of tokens 2t, 2t+1 at 16i+g, the same at 16i+8+g}
constexpr int kRecA = kRecK + 8 * 128;   // [8][4 t]{e(16i+2t), e(16i+2t+1), e(16i+8+2t), e(16i+8+2t+1)}
constexpr int kRecP = kRecA + 128;       // [32]{P(g,2t), P(g,2t+1)}
constexpr int kRecV = kRecP + 64;        // [8 tiles of columns][32]{V of tokens 2t, 2t+1 at 16i+g, at 16i+8+g}
constexpr int kRecFloats = kRecV + 8 * 128;

// A CTA per head and block of tokens, a thread per d.  Reads 6 x 512 bytes a token-head (fp32), writes 2.1 KB
// that are read back from L2; bound by its instructions (1200 a thread, half of them the Gram sums and
// their addresses) and the loads' latency.  Measured: 24576 token-heads 30 us (2.5 TB/s of inputs).  Tokens past the sequence's end become no-ops
// (gate 1, zeros elsewhere).
template <class T>
__global__ void __launch_bounds__(kD, 4) rec_prep_kernel(RecParams p, float* rec, int tok0, int nblk) {
  __shared__ float part[kD / 32][64];
  __shared__ float lp[64];                  // L_ts in 8 t + s (s < t), P_ts in 8 s + t (s <= t)
  __shared__ __align__(16) float xm[8][8];  // X
  const int d = threadIdx.x, lane = d & 31, warp = d >> 5;
  const int bh = blockIdx.x / nblk, blk = blockIdx.x % nblk;
  const int b = bh / p.H, h = bh % p.H;
  const int t0 = tok0 + blk * kTok, left = valid_len(p, b, false) - t0;
  if (left <= 0) return;
  float* out = rec + (size_t)blockIdx.x * kRecFloats;
  float q[kTok], k[kTok], bk[kTok], a[kTok], v[kTok], wv[kTok];
  {
    const void* base[6] = {p.q, p.k, p.v, p.w, p.b, p.g};
    const T* src[6];
    int sl[6];  // a block's tokens are within 32 bits of one another (checked by the entry)
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      src[i] = static_cast<const T*>(base[i]) + b * p.sb[i] + h * p.sh[i] + t0 * p.sl[i] + d;
      sl[i] = (int)p.sl[i];
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {  // all of the loads first; the last valid token stands in for those past it
      const int tt = min(t, left - 1);
      q[t] = ld1(src[0] + tt * sl[0]);
      k[t] = ld1(src[1] + tt * sl[1]);
      v[t] = ld1(src[2] + tt * sl[2]);
      wv[t] = ld1(src[3] + tt * sl[3]);
      bk[t] = ld1(src[4] + tt * sl[4]);
      a[t] = ld1(src[5] + tt * sl[5]);
    }
  }
  bool positive = false;
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    const bool on = t < left;
    positive |= a[t] > 0.f;
    a[t] = on ? expf(a[t] > 0.f ? 0.f : a[t]) : 1.f;  // a NaN stays one
    q[t] = on ? q[t] * p.scale : 0.f;
    k[t] = on ? k[t] : 0.f;
    bk[t] = on ? bk[t] * k[t] : 0.f;
    wv[t] = on ? wv[t] * v[t] : 0.f;
  }
  if (positive) p.flags[0] = 1u;
  float gram[64], kh[kTok];
#pragma unroll
  for (int s = 0; s < kTok; ++s) {
    float c = k[s];
    gram[9 * s] = q[s] * c;
#pragma unroll
    for (int t = s + 1; t < kTok; ++t) {
      c *= a[t];
      gram[8 * t + s] = bk[t] * c;
      gram[8 * s + t] = q[t] * c;
    }
    kh[s] = c;  // k_s e^{G_8 - G_s}
  }
  // 64 sums over the warp's lanes, halving: lane l ends with entries 2 l and 2 l + 1
#pragma unroll
  for (int half = 32; half >= 2; half >>= 1) {
    const bool up = lane & (half >> 1);
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float keep = up ? gram[i + half] : gram[i], give = up ? gram[i] : gram[i + half];
      gram[i] = keep + __shfl_xor_sync(0xffffffffu, give, half >> 1);
    }
  }
  *reinterpret_cast<float2*>(&part[warp][2 * lane]) = make_float2(gram[0], gram[1]);
  __syncthreads();
  if (d < 64) lp[d] = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
  __syncthreads();
  if (d < 8) {  // column d of X by forward substitution
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = i == d ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) y[i] = fmaf(-lp[8 * i + j], y[j], y[i]);
      xm[i][d] = y[i];
    }
  }
  // what needs no X, meanwhile.  Two lanes hold the two halves of 16 bytes of the record: each takes every
  // second piece.
  const bool odd = d & 1, high = d & 8;
  float e = 1.f, be[kTok], qe[kTok];
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    e *= a[t];
    be[t] = bk[t] * e;
    qe[t] = q[t] * e;
  }
  out[kRecA + ((d >> 4) * 4 + ((d & 7) >> 1)) * 4 + ((d >> 3) & 1) * 2 + (d & 1)] = e;
  const int at = (d >> 4) * 32 + (d & 7) * 4 + (high ? 2 : 0);
#pragma unroll
  for (int t = 0; t < 4; t += 2) {
    const float k0 = __shfl_xor_sync(0xffffffffu, high ? kh[t] : kh[t + 4], 8);
    const float k1 = __shfl_xor_sync(0xffffffffu, high ? kh[t + 1] : kh[t + 5], 8);
    reinterpret_cast<float4*>(out + kRecK)[at + (t >> 1)] =
        high ? make_float4(k0, k1, kh[t + 4], kh[t + 5]) : make_float4(kh[t], kh[t + 1], k0, k1);
  }
  if (d < 64) {
    const int l = d >> 1, g = l >> 2, s = (l & 3) * 2 + (d & 1);
    out[kRecP + d] = s <= g ? lp[8 * s + g] : 0.f;
  }
  __syncthreads();
  float bx[kTok], vx[kTok];
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    bx[t] = be[t];
    vx[t] = wv[t];
#pragma unroll
    for (int s = 0; s < t; ++s) {
      bx[t] = fmaf(xm[t][s], be[s], bx[t]);
      vx[t] = fmaf(xm[t][s], wv[s], vx[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < kTok; t += 2) {
    const float bo = __shfl_xor_sync(0xffffffffu, odd ? bx[t] : bx[t + 1], 1);
    const float qo = __shfl_xor_sync(0xffffffffu, odd ? qe[t] : qe[t + 1], 1);
    reinterpret_cast<float4*>(out + kRecDot)[(d >> 3) * 32 + (t + odd) * 4 + ((d & 7) >> 1)] =
        odd ? make_float4(bo, bx[t + 1], qo, qe[t + 1]) : make_float4(bx[t], bo, qe[t], qo);
  }
#pragma unroll
  for (int t = 0; t < 4; t += 2) {
    const float v0 = __shfl_xor_sync(0xffffffffu, high ? vx[t] : vx[t + 4], 8);
    const float v1 = __shfl_xor_sync(0xffffffffu, high ? vx[t + 1] : vx[t + 5], 8);
    reinterpret_cast<float4*>(out + kRecV)[at + (t >> 1)] =
        high ? make_float4(v0, v1, vx[t + 4], vx[t + 5]) : make_float4(vx[t], vx[t + 1], v0, v1);
  }
}

// x = hi + lo: hi is x in tf32, rounded to nearest, and the tensor instruction drops the 13 low bits
// of lo, 2^-21 of x at most and either way.  A NaN may lose its bits in hi but stays one in lo.
struct Split { uint32_t hi, lo; };
__device__ __forceinline__ Split split(float x) {
  Split s;
  s.hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  s.lo = __float_as_uint(x - __uint_as_float(s.hi));
  return s;
}
struct SplitA { uint32_t hi[4], lo[4]; };
// An accumulator tile as the next product's first operand (k = t and t + 4 are columns 2t and 2t + 1).
__device__ __forceinline__ SplitA split_tile(const float c[4]) {
  SplitA a;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Split s = split(c[(i & 1) * 2 + (i >> 1)]);
    a.hi[i] = s.hi;
    a.lo[i] = s.lo;
  }
  return a;
}
__device__ __forceinline__ void mma1688(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// lo hi and hi lo into one accumulator, hi hi into another
__device__ __forceinline__ void mma3(float big[4], float small[4], const SplitA& a, float b0, float b1) {
  const Split x = split(b0), y = split(b1);
  mma1688(small, a.lo, x.hi, y.hi);
  mma1688(big, a.hi, x.hi, y.hi);
  mma1688(small, a.hi, x.lo, y.lo);
}

// What both forms of the kernel share.
struct SeqSpan {
  int n, blocks;     // valid tokens of this launch, and their blocks
  long long state;   // element offset of the head's state, negative for zeros
  float* o;          // outputs of the launch's first token, at the CTA's first column
};
template <int kThreads, int kCols>
__device__ __forceinline__ SeqSpan seq_span(const RecParams& p, int tok0, int nblk, bool first) {
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, tid = threadIdx.x;
  const bool report = first && tid == 0 && h == 0 && blockIdx.y == 0;
  SeqSpan r;
  r.n = max(0, min(valid_len(p, b, report) - tok0, nblk * kTok));
  r.blocks = (r.n + kTok - 1) / kTok;
  r.o = p.o + b * p.ob + h * p.oh + tok0 * p.ol + blockIdx.y * kCols;
  const int end = min(p.L - tok0, nblk * kTok);
  for (int i = r.n * kCols + tid; i < end * kCols; i += kThreads)  // past the sequence's end
    r.o[(i / kCols) * p.ol + i % kCols] = 0.f;
  r.state = bh;
  if (first) {
    const int row = state_row(p, b, report);
    r.state = row < 0 ? -1 : (long long)row * p.H + h;
  }
  r.state *= kD * kD;
  return r;
}
// Tile j of a warp: columns g (entries 0, 1) and g + 8 (2, 3), rows 8 j + 2 t and 8 j + 2 t + 1.
template <int kJ>
__device__ __forceinline__ void seq_load(float s[kJ][4], const float* state, const SeqSpan& r, size_t mine) {
#pragma unroll
  for (int j = 0; j < kJ; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      s[j][c] = r.state >= 0 ? state[r.state + mine + (j * 8 + (c & 1)) * kD + (c >> 1) * 8] : 0.f;
}
template <int kJ>
__device__ __forceinline__ void seq_store(const float s[kJ][4], const RecParams& p, size_t mine, bool last) {
  float* to = p.h_out + (size_t)blockIdx.x * (kD * kD) + mine;
#pragma unroll
  for (int j = 0; j < kJ; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      to[(j * 8 + (c & 1)) * kD + (c >> 1) * 8] = last ? sanitize(s[j][c], p.clip) : s[j][c];
}
// The launch's tokens by the definition, for 16 columns from `col` on (the CTA's column `mine`), by the CTA's first
// four warps: a thread has 16 rows of a column.  The state has not been written back yet, and the records are done
// with: 19 KB of their place are used.  Measured: 0.6 us a token (the latency of its loads and barriers).
constexpr int kLitThreads = 128;
template <class T>
__device__ __noinline__ void seq_literal(const RecParams& p, const SeqSpan& r, const float* state, int tok0, int col,
                                         int mine, bool last) {
  extern __shared__ float4 smem4[];
  float* mem = reinterpret_cast<float*>(smem4);
  const int tid = threadIdx.x, c = tid & 15, d0 = (tid >> 4) * 16, warp = tid >> 5, row = tid >> 4;
  const long long b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  float (*vec)[4][kD] = reinterpret_cast<float (*)[4][kD]>(mem);  // a, k, b k, q of a token
  float (*wv)[16] = reinterpret_cast<float (*)[16]>(mem + kTok * 4 * kD);
  float (*part)[4][16] = reinterpret_cast<float (*)[4][16]>(mem + kTok * (4 * kD + 16));  // by a token's parity
  float (*outs)[4][16] = part + 2;                                                        // by token
  auto barrier = [] { asm volatile("bar.sync 2, %0;" ::"n"(kLitThreads) : "memory"); };
  auto in = [&](const void* x, int i, int t, int d) {
    return ld1(static_cast<const T*>(x) + b * p.sb[i] + h * p.sh[i] + (tok0 + t) * p.sl[i] + d);
  };
  const size_t at = (size_t)d0 * kD + col + c;
  float s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = r.state >= 0 ? state[r.state + at + i * kD] : 0.f;
  for (int t0 = 0; t0 < r.n; t0 += kTok) {
    const int n = min(kTok, r.n - t0);
    float x[kTok][4];
#pragma unroll
    for (int t = 0; t < kTok; ++t) {  // all of the loads first; the last token stands in for those past it
      const int tt = t0 + min(t, n - 1);
      x[t][0] = in(p.g, 5, tt, tid);
      x[t][1] = in(p.k, 1, tt, tid);
      x[t][2] = in(p.b, 4, tt, tid);
      x[t][3] = in(p.q, 0, tt, tid);
    }
    barrier();  // the tokens before are done with
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      vec[t][0][tid] = expf(x[t][0] > 0.f ? 0.f : x[t][0]);
      vec[t][1][tid] = x[t][1];
      vec[t][2][tid] = x[t][2] * x[t][1];
      vec[t][3][tid] = x[t][3];
    }
    if (row < n) wv[row][c] = in(p.w, 3, t0 + row, col + c) * in(p.v, 2, t0 + row, col + c);
    barrier();
    for (int t = 0; t < n; ++t) {
      float sum = 0.f, out = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] *= vec[t][0][d0 + i];
        sum = fmaf(vec[t][2][d0 + i], s[i], sum);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if ((tid & 16) == 0) part[t & 1][warp][c] = sum;
      barrier();
      const float d = wv[t][c] - ((part[t & 1][0][c] + part[t & 1][1][c]) + (part[t & 1][2][c] + part[t & 1][3][c]));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = fmaf(vec[t][1][d0 + i], d, s[i]);
        out = fmaf(vec[t][3][d0 + i], s[i], out);
      }
      out += __shfl_xor_sync(0xffffffffu, out, 16);
      if ((tid & 16) == 0) outs[t][warp][c] = out;
    }
    barrier();
    if (row < n)
      r.o[(t0 + row) * p.ol + mine + c] =
          sanitize(p.scale * ((outs[row][0][c] + outs[row][1][c]) + (outs[row][2][c] + outs[row][3][c])), p.clip);
  }
  float* to = p.h_out + (size_t)blockIdx.x * (kD * kD) + at;
#pragma unroll
  for (int i = 0; i < 16; ++i) to[i * kD] = last ? sanitize(s[i], p.clip) : s[i];
}
__device__ __forceinline__ void seq_again(const RecParams& p, const SeqSpan& r, const float* state, int tok0, int col,
                                          int mine, bool last) {
  if (p.bf16) seq_literal<__nv_bfloat16>(p, r, state, tok0, col, mine, last);
  else seq_literal<float>(p, r, state, tok0, col, mine, last);
}
__device__ __forceinline__ float not_finite4(const float x[4]) {
  return (not_finite(x[0]) + not_finite(x[1])) + (not_finite(x[2]) + not_finite(x[3]));
}
// o + P d, stored for the block's valid tokens.  `pm`: the record's P.
__device__ __forceinline__ void seq_out(const RecParams& p, const SeqSpan& r, int blk, int col, const float o[4],
                                        const SplitA& d, const float* pm) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const float2 f = *reinterpret_cast<const float2*>(pm + lane * 2);
  float big[4] = {}, small[4] = {};
  mma3(big, small, d, f.x, f.y);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int tok = blk * kTok + 2 * t + (c & 1);
    if (tok < r.n) r.o[tok * p.ol + col + (c >> 1) * 8] = sanitize(o[c] + (big[c] + small[c]), p.clip);
  }
}
template <int kJ>
__device__ __forceinline__ void seq_update(float s[kJ][4], const SplitA& d, const float* slot, int j0, int lane) {
#pragma unroll
  for (int j = 0; j < kJ; j += 2) {
    const float4 kk = *reinterpret_cast<const float4*>(slot + kRecK + ((j0 + j) * 16 + lane) * 4);
    const float4 e = *reinterpret_cast<const float4*>(slot + kRecA + ((j0 + j) * 2 + (lane & 3)) * 4);
    float ub[2][4] = {}, us[2][4] = {};
    mma3(ub[0], us[0], d, kk.x, kk.y);
    mma3(ub[1], us[1], d, kk.z, kk.w);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s[j][c] = fmaf(c & 1 ? e.y : e.x, s[j][c], ub[0][c] + us[0][c]);
      s[j + 1][c] = fmaf(c & 1 ? e.w : e.z, s[j + 1][c], ub[1][c] + us[1][c]);
    }
  }
}
__device__ __forceinline__ float4 lds4(const float* p) { return *reinterpret_cast<const float4*>(p); }
// The records' way into the ring: bulk copies that one thread issues, a barrier object per slot.  Waits
// give up after the library's limit, tell the host and do not wait again; the thread that issued the copies
// issues no more then, and gives those on their way one more limit each before the CTA ends (drain).
template <int kSlots>
struct SeqRing {
  uint64_t* bars;
  uint32_t* flags;
  int* last;  // in shared memory: blocks that had been issued when the thread that issues them gave up
  bool gave_up = false;
  __device__ void init() {  // one thread
    for (int i = 0; i < kSlots; ++i) mbar_init(bars + i, 1);
    fence_mbar_init();
  }
  __device__ void fetch(int blk, float* dst, const float* from, int v_from, int v_floats) {  // one thread
    const int slot = blk % kSlots;
    mbar_arrive_expect_tx(bars + slot, (kRecV + v_floats) * 4);
    bulk_g2s(dst, from, kRecV * 4, bars + slot);
    bulk_g2s(dst + kRecV, from + kRecV + v_from, v_floats * 4, bars + slot);
  }
  __device__ void wait(int slot, uint32_t parity, int issued) {  // `issued`: blocks by now, 0 by other threads
    if (gave_up || mbar_try_wait(bars + slot, parity)) return;
    const long long t0 = clock64();
    while (!mbar_try_wait(bars + slot, parity)) {
      if (clock64() - t0 > kWaitCycles) {
        gave_up = true;
        flags[2] = 1u;
        if (issued) *last = issued;
        return;
      }
    }
  }
  __device__ void drain(int blocks) {  // the thread that fetches
    if (!gave_up) return;
    const int end = min(*last, blocks);
    for (int blk = max(0, end - kSlots); blk < end; ++blk) {
      const long long t0 = clock64();
      while (!mbar_try_wait(bars + blk % kSlots, (blk / kSlots) & 1) && clock64() - t0 <= kWaitCycles) {
      }
    }
  }
};

// Many heads: a warp owns 16 columns and all of d, a CTA kCT such tiles.  Bound by the tensor pipe (144
// products of 8 cycles a warp and block, half busy) and the splits' integer slots.  Measured: 384 heads x 80
// tokens 72 us, 11 us of it the floor of its bytes.  The records arrive through a ring.  The bound of
// three CTAs an SM gives a thread 168 registers; without it the compiler takes 128 and spills (75 us).
template <int kCT>
__global__ void __launch_bounds__(kCT * 32, 3) rec_wide_kernel(const __grid_constant__ RecParams p, const float* rec,
                                                               const float* state, int tok0, int nblk, bool first,
                                                               bool last) {
  constexpr int kThreads = kCT * 32, kSlots = 3, kSlot = kRecV + kCT * 128;
  extern __shared__ float4 smem4[];
  __shared__ uint64_t bars[kSlots];
  __shared__ int issued;
  float* smem = reinterpret_cast<float*>(smem4);
  const int tid = threadIdx.x, lane = tid & 31, ct = tid >> 5, g = lane >> 2, t = lane & 3;
  const SeqSpan r = seq_span<kThreads, kCT * 16>(p, tok0, nblk, first);
  if (r.blocks == 0 && !first && !last) return;
  const size_t mine = (size_t)(2 * t) * kD + (blockIdx.y * kCT + ct) * 16 + g;
  float s[16][4];
  seq_load<16>(s, state, r, mine);
  const float* src = rec + (size_t)blockIdx.x * nblk * kRecFloats;
  SeqRing<kSlots> ring{bars, p.flags, &issued};
  if (tid == 0) ring.init();
  __syncthreads();
  auto fetch = [&](int blk) {
    if (tid == 0 && blk < r.blocks && !ring.gave_up)
      ring.fetch(blk, smem + (blk % kSlots) * kSlot, src + (size_t)blk * kRecFloats, blockIdx.y * kCT * 128, kCT * 128);
  };
#pragma unroll
  for (int i = 0; i < kSlots - 1; ++i) fetch(i);
  float probe = 0.f;
  for (int blk = 0; blk < r.blocks; ++blk) {
    ring.wait(blk % kSlots, (blk / kSlots) & 1, tid == 0 ? blk + kSlots - 1 : 0);
    __syncthreads();          // every warp is done with block blk - 1
    fetch(blk + kSlots - 1);  // into that block's slot
    const float* slot = smem + (blk % kSlots) * kSlot;
    float rr[4], o[4];
    {
      float rb[2][4] = {}, rs[4] = {}, ob[2][4] = {}, os[4] = {};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float4 f = lds4(slot + kRecDot + (j * 32 + lane) * 4);
        const SplitA a = split_tile(s[j]);
        mma3(rb[j & 1], rs, a, f.x, f.y);
        mma3(ob[j & 1], os, a, f.z, f.w);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        rr[c] = (rb[0][c] + rb[1][c]) + rs[c];
        o[c] = (ob[0][c] + ob[1][c]) + os[c];
      }
    }
    const float4 v = lds4(slot + kRecV + (ct * 32 + lane) * 4);
    const float dl[4] = {v.x - rr[0], v.y - rr[1], v.z - rr[2], v.w - rr[3]};
    const SplitA d = split_tile(dl);
    probe += not_finite4(dl) + not_finite4(o);
    seq_out(p, r, blk, ct * 16 + g, o, d, slot + kRecP);
    seq_update<16>(s, d, slot, 0, lane);
  }
  if (tid == 0) ring.drain(r.blocks);
  static_assert(kThreads == kLitThreads);
  if (!__syncthreads_or(probe != 0.f)) {
    seq_store<16>(s, p, mine, last);
  } else {
    for (int i = 0; i < kCT; ++i) seq_again(p, r, state, tok0, (blockIdx.y * kCT + i) * 16, i * 16, last);
  }
}

// Few heads, where a block's chain of dependent steps is what counts (measured: 422 ns for 8 tokens, 6 heads
// x 4096 tokens 216 us): kW warps share 16 columns and take 16 / kW tiles of d each; one more warp sees to the
// records and one finishes the outputs, a block behind.  Two CTAs fit on an SM by shared memory; the bound
// of three is for registers (96 a thread; without it the compiler takes 80, and 265 us).  One barrier per
// block: before it the partial sums r of the block are written, after it every warp adds them up.  What is
// double-buffered by the block's parity:
//   rpart  written before barrier blk, read until barrier blk + 1
//   opart, delta  written after barrier blk, read between barriers blk + 1 and blk + 2
template <int kW>
__global__ void __launch_bounds__((kW + 2) * 32, 3) rec_deep_kernel(const __grid_constant__ RecParams p,
                                                                    const float* rec, const float* state, int tok0,
                                                                    int nblk, bool first, bool last) {
  constexpr int kThreads = (kW + 2) * 32, kJ = 16 / kW, kSlots = 6, kSlot = kRecV + 128;
  extern __shared__ float4 smem4[];
  float* smem = reinterpret_cast<float*>(smem4);
  float4* rpart = smem4 + kSlots * kSlot / 4;  // [2][kW][32]
  float4* opart = rpart + 2 * kW * 32;         // [2][kW][32]
  float4* delta = opart + 2 * kW * 32;         // [2][32]
  __shared__ uint64_t bars[kSlots];
  __shared__ int issued;
  __shared__ int bad;  // set before the last barrier, where a warp has met a value that is not finite
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const SeqSpan r = seq_span<kThreads, 16>(p, tok0, nblk, first);
  if (r.blocks == 0 && !first && !last) return;
  auto barrier = [] { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); };
  if (warp == kW) {  // copies
    const float* src = rec + (size_t)blockIdx.x * nblk * kRecFloats;
    SeqRing<kSlots> ring{bars, p.flags, &issued};
    if (lane == 0) {
      ring.init();
      bad = 0;
    }
    __syncwarp();
    auto fetch = [&](int blk) {
      if (lane == 0 && blk < r.blocks && !ring.gave_up)
        ring.fetch(blk, smem + (blk % kSlots) * kSlot, src + (size_t)blk * kRecFloats, blockIdx.y * 128, 128);
    };
    auto landed = [&](int blk) {
      if (blk < r.blocks) ring.wait(blk % kSlots, (blk / kSlots) & 1, lane ? 0 : blk ? blk + kSlots - 3 : kSlots - 2);
    };
    for (int i = 0; i < kSlots - 2; ++i) fetch(i);
    landed(0);
    barrier();  // block 0 is here
    for (int blk = 0; blk < r.blocks; ++blk) {
      landed(blk + 1);
      barrier();                // block blk + 1 is here, and every warp is done with block blk - 2
      fetch(blk + kSlots - 2);  // into that block's slot
    }
    if (lane == 0) ring.drain(r.blocks);
    barrier();
    return;
  }
  if (warp == kW + 1) {  // outputs
    barrier();
    for (int blk = 0; blk < r.blocks; ++blk) {
      barrier();  // barrier blk: block blk - 1 is ready
      if (blk == 0) continue;
      const int par = (blk - 1) & 1;
      float o[4] = {};
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const float4 x = opart[(par * kW + i) * 32 + lane];
        o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w;
      }
      const float4 x = delta[par * 32 + lane];
      const float dl[4] = {x.x, x.y, x.z, x.w};
      seq_out(p, r, blk - 1, g, o, split_tile(dl), smem + ((blk - 1) % kSlots) * kSlot + kRecP);
    }
    barrier();
    if (r.blocks && !bad) {
      const int blk = r.blocks - 1, par = blk & 1;
      float o[4] = {};
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const float4 x = opart[(par * kW + i) * 32 + lane];
        o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w;
      }
      const float4 x = delta[par * 32 + lane];
      const float dl[4] = {x.x, x.y, x.z, x.w};
      seq_out(p, r, blk, g, o, split_tile(dl), smem + (blk % kSlots) * kSlot + kRecP);
    }
    return;
  }
  const int j0 = warp * kJ;
  const size_t mine = (size_t)(8 * j0 + 2 * t) * kD + blockIdx.y * 16 + g;
  float s[kJ][4];
  seq_load<kJ>(s, state, r, mine);
  float probe = 0.f;
  barrier();
  for (int blk = 0; blk < r.blocks; ++blk) {
    const float* slot = smem + (blk % kSlots) * kSlot;
    const int par = blk & 1;
    SplitA a[kJ];
    float4 f[kJ];
    float big[2][4] = {}, small[2][4] = {};
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      f[j] = lds4(slot + kRecDot + ((j0 + j) * 32 + lane) * 4);
      a[j] = split_tile(s[j]);
      mma3(big[j & 1], small[j & 1], a[j], f[j].x, f[j].y);
    }
    rpart[(par * kW + warp) * 32 + lane] =
        make_float4((big[0][0] + big[1][0]) + (small[0][0] + small[1][0]), (big[0][1] + big[1][1]) + (small[0][1] + small[1][1]),
                    (big[0][2] + big[1][2]) + (small[0][2] + small[1][2]), (big[0][3] + big[1][3]) + (small[0][3] + small[1][3]));
    float ob[2][4] = {}, os[2][4] = {};
#pragma unroll
    for (int j = 0; j < kJ; ++j) mma3(ob[j & 1], os[j & 1], a[j], f[j].z, f[j].w);
    barrier();
    const float4 v = lds4(slot + kRecV + lane * 4);
    float rr[4] = {};
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      const float4 x = rpart[(par * kW + i) * 32 + lane];
      rr[0] += x.x; rr[1] += x.y; rr[2] += x.z; rr[3] += x.w;
    }
    const float dl[4] = {v.x - rr[0], v.y - rr[1], v.z - rr[2], v.w - rr[3]};
    const SplitA d = split_tile(dl);
    seq_update<kJ>(s, d, slot, j0, lane);
    const float o[4] = {(ob[0][0] + ob[1][0]) + (os[0][0] + os[1][0]), (ob[0][1] + ob[1][1]) + (os[0][1] + os[1][1]),
                        (ob[0][2] + ob[1][2]) + (os[0][2] + os[1][2]), (ob[0][3] + ob[1][3]) + (os[0][3] + os[1][3])};
    opart[(par * kW + warp) * 32 + lane] = make_float4(o[0], o[1], o[2], o[3]);
    probe += not_finite4(dl) + not_finite4(o);
    if (warp == 0) delta[par * 32 + lane] = make_float4(dl[0], dl[1], dl[2], dl[3]);
  }
  if (probe != 0.f) bad = 1;
  barrier();
  static_assert(kW * 32 == kLitThreads);
  if (!bad) seq_store<kJ>(s, p, mine, last);
  else seq_again(p, r, state, tok0, blockIdx.y * 16, 0, last);
}

template <class K>
cudaError_t launch_seq(K kernel, int cols, int threads, int bytes, const RecParams& p, const float* rec, int BH,
                       int tok0, int nblk, bool first, bool last, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(BH, kD / cols), threads, bytes, st>>>(p, rec, first ? p.h0 : p.h_out, tok0, nblk, first, last);
  return cudaGetLastError();
}
template <int kCT>
cudaError_t launch_wide(const RecParams& p, const float* rec, int BH, int tok0, int nblk, bool first, bool last,
                        cudaStream_t st) {
  return launch_seq(rec_wide_kernel<kCT>, kCT * 16, kCT * 32, 3 * (kRecV + kCT * 128) * 4, p, rec, BH, tok0, nblk,
                    first, last, st);
}
template <int kW>
cudaError_t launch_deep(const RecParams& p, const float* rec, int BH, int tok0, int nblk, bool first, bool last,
                        cudaStream_t st) {
  return launch_seq(rec_deep_kernel<kW>, 16, (kW + 2) * 32, 6 * (kRecV + 128) * 4 + (4 * kW + 2) * 512, p, rec, BH,
                    tok0, nblk, first, last, st);
}

// Blocks of tokens that one pair of launches covers: as many as keep the records within 64 MiB
// (they are read back from L2), but eight at least, so that the state's own traffic stays small.
int seg_blocks(long long BH, int L) {
  const long long fit = (64LL << 20) / (BH * kRecFloats * 4), all = ((long long)L + kTok - 1) / kTok;
  const long long n = fit < 8 ? 8 : fit;
  return (int)(n < all ? n : all);
}

template <class T>
cudaError_t launch(const RecParams& p, int BH, float* rec, cudaStream_t st) {
  if (p.L <= 1) {
    rec_step_kernel<T><<<BH, kStepThreads, 0, st>>>(p);
    return cudaGetLastError();
  }
  const int seg = seg_blocks(BH, p.L);
  // Four warps on a head's 16 columns shorten a block's chain but repeat part of its work; measured on
  // the device (fp32, deep / wide): 6 heads x 4096 tokens 250 / 663 us, 48 x 1024 205 / 226, 96 x 777
  // 308 / 314, 108 x 400 169 / 170, 120 x 400 192 / 177, 192 x 256 198 / 176, 384 x 192 310 / 264.  Where
  // the two meet the deep form's 8 CTAs a head, two to an SM, take three turns.
  const bool deep = (long long)BH * 8 <= 6LL * kSmCount;
  for (int t0 = 0; t0 < p.L; t0 += seg * kTok) {
    const int nblk = min(seg, (p.L - t0 + kTok - 1) / kTok);
    const bool first = t0 == 0, last = t0 + seg * kTok >= p.L;
    rec_prep_kernel<T><<<BH * nblk, kD, 0, st>>>(p, rec, t0, nblk);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = deep ? launch_deep<4>(p, rec, BH, t0, nblk, first, last, st)
             : launch_wide<4>(p, rec, BH, t0, nblk, first, last, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Grids count heads x blocks of tokens along x.
gdn2_status check_rec(const gdn2_rec_desc* d) {
  if (!d || d->B <= 0 || d->H <= 0 || d->L < 0 || d->D <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->in_dtype != GDN2_F32 && d->in_dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (!(d->clip > 0.f) || (int64_t)d->B * d->H > (1 << 26)) return GDN2_ERR_INVALID_ARGUMENT;
  return d->D == kD && d->L <= (1 << 30) ? GDN2_OK : GDN2_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_recurrent_workspace_bytes(const gdn2_rec_desc* d) {
  using namespace gdn2;
  if (check_rec(d) != GDN2_OK || d->L <= 1) return 0;
  return (size_t)d->B * d->H * seg_blocks((long long)d->B * d->H, d->L) * kRecFloats * 4;
}

extern "C" gdn2_status gdn2_recurrent(const gdn2_rec_desc* d, const void* q, const void* k, const void* v,
                                      const void* w, const void* b, const void* g, const float* h0,
                                      const int32_t* h_index, const int32_t* lengths, float* o, float* h_out,
                                      void* workspace, uint32_t* flags, void* stream) {
  using namespace gdn2;
  const gdn2_status status = check_rec(d);
  if (status != GDN2_OK) return status;
  if (d->L > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))) return GDN2_ERR_INVALID_ARGUMENT;
  const int el = d->in_dtype == GDN2_BF16 ? 2 : 4;
  const void* ins[6] = {q, k, v, w, b, g};
  RecParams p{};
  if (d->L > 0) {
    for (int i = 0; i < 6; ++i) {
      if (!ins[i] || !aligned16(ins[i])) return GDN2_ERR_INVALID_ARGUMENT;
      for (int j = 0; j < 3; ++j)
        if (d->stride[i][j] < 0 || (d->stride[i][j] * el) % 16) return GDN2_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 6; ++i)
      if (d->stride[i][2] >= 1 << 27) return GDN2_ERR_INVALID_ARGUMENT;
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
  p.bf16 = el == 2;
  p.scale = d->scale; p.clip = d->clip;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* rec = static_cast<float*>(workspace);
  const cudaError_t e = el == 2 ? launch<__nv_bfloat16>(p, d->B * d->H, rec, st) : launch<float>(p, d->B * d->H, rec, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
