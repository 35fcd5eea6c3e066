// One AdamW step over all tensors of a model (sm_100a), with the gradients' global norm, clipping by it and a
// guard that skips steps whose loss or norm is not finite or whose norm jumps.
//   n = |g|,  g' = g clip / max(n, clip)
//   m = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// In the moments each operation is rounded to fp32 by itself, in this order, and so is the root that is stored in
// 8 bits: codes depend on every bit, and these do not depend on how a compiler joins products and sums.  The
// squares of the norm are summed in fp64 in a fixed order.
//
// Moments in 8 bits: 256 neighbouring values share a scale.  m is e4m3 of m / scale, scale = max |m| / 448.  Of v
// the root r is stored, unsigned with four bits of exponent and four of mantissa (c 2^-18 below code 16, else
// (16 + c % 16) 2^(c / 16 - 19)), scale = max r / 1.9375: half a step is 1/32 of r.  A root above zero is never
// stored as zero, or a later step would divide by eps alone.
//
// Bytes bound it: the gradients are read once for their norm and once for the update, p, m and v are read and
// written once.  Two launches: the norm's, whose last CTA also counts the steps and prepares the tensors'
// factors, and the update's.  The tensors' table travels in the kernels' parameters: nothing is copied to the
// device, and a captured graph keeps what it needs.
//
// Measured, 39 M fp32 weights: norm 39 us (156 MB; the last CTA's turn is some 6 us of it), update 161 us (1095 MB at 6.8
// TB/s); with 8-bit moments 125 us (626 MB: 64 instructions a value, two thirds of the issue slots).  348 M bf16 weights with
// 8-bit moments: 940 us (3.5 GB).
#include <cuda_fp8.h>

#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

constexpr int kChunk = 8192;          // values of a tensor that a CTA takes at a time
constexpr int kBlock = 256;           // values that share a scale
constexpr int kAdamThreads = 256;
constexpr float kNormal = 1.17549435e-38f;

struct AdamEntry {
  void *p, *m, *v;
  const void* g;
  float *ms, *vs, *step;
  const float* lr_at;
  double lr, wd;
  long long n;
  int first;                          // the tensor's first chunk
  short bf16, vec;                    // types of p and g; whether all of it may be read 4 values at a time
};
template <int N>
struct AdamTable {
  AdamEntry e[N];
  int count, chunks;
};
struct Factors {                      // of a tensor
  float size, root, decay;            // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
};
struct AdamControl {                  // the caller's control words
  float ema, norm, ok, coef;
  unsigned ticket;
};
struct AdamParams {
  AdamControl* ctl;
  double* parts;                      // workspace: a CTA's sum of squares
  Factors* factors;                   // workspace: a tensor's factors
  const float* loss;
  double b1, b2, log2_b1, log2_b2;
  float fb1, gb1, fb2, gb2, eps, clip, spike;
  int norm, part0, all_parts, tensor0, alone;
};

template <int N>
__device__ __forceinline__ int find(const AdamTable<N>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The factors of the tensors' next step, and once the guard has decided for it the step counts.
template <int N>
__device__ __forceinline__ void factors(const AdamTable<N>& t, const AdamParams& a) {
  for (int i = threadIdx.x; i < t.count; i += blockDim.x) {
    const AdamEntry& e = t.e[i];
    const double n = *e.step + 1.f, lr = e.lr_at ? (double)*e.lr_at : e.lr;
    a.factors[a.tensor0 + i] = {(float)(lr / (1.0 - exp2(n * a.log2_b1))), (float)rsqrt(1.0 - exp2(n * a.log2_b2)),
                                (float)(1.0 - lr * e.wd)};
  }
}
template <int N>
__device__ __forceinline__ void count_up(const AdamTable<N>& t) {
  for (int i = threadIdx.x; i < t.count; i += blockDim.x) *t.e[i].step += 1.f;
}

__device__ __forceinline__ double block_sum(double s, double* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < kAdamThreads / 32; ++i) s += sm[i];
  __syncthreads();
  return s;
}

// |x| in fp64, put together from x's bits: the conversion instruction runs at a fraction of the rate.  The bits
// stand for |x| 2^-896 for every finite x; an infinity or a NaN becomes 2^128 or more, and the norm infinite.
__device__ __forceinline__ double wide(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return __hiloint2double((int)(u >> 3), (int)(u << 29)) * 0x1p896;
}
template <class T>
__device__ __forceinline__ void squares(const T* g, int n, bool vec, double q[4]) {
  int done = 0;
  if (vec) {
    float v[kChunk / 4 / kAdamThreads][4];
#pragma unroll
    for (int i = 0; i < kChunk / 4 / kAdamThreads; ++i) {
      const int at = 4 * (i * kAdamThreads + (int)threadIdx.x);
      if (at + 4 <= n) ld4(g + at, v[i]);
      else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kChunk / 4 / kAdamThreads; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double w = wide(v[i][j]);
        q[j] = fma(w, w, q[j]);
      }
    done = n & ~3;
  }
  for (int i = done + threadIdx.x; i < n; i += kAdamThreads) {
    const double v = wide(ld1(g + i));
    q[0] = fma(v, v, q[0]);
  }
}

// Sums of the gradients' squares; the last CTA adds the CTAs' up and decides.
template <int N>
__global__ void __launch_bounds__(kAdamThreads) adamw_norm_kernel(const __grid_constant__ AdamTable<N> t,
                                                                  const __grid_constant__ AdamParams a) {
  __shared__ double sm[kAdamThreads / 32];
  __shared__ bool final, go;
  pdl_enter();
  double total = 0.0;
  if (a.alone && blockIdx.x == gridDim.x - 1) factors(t, a);  // the last CTA to start has the least to add up
  if (a.norm) {
    double q[4] = {};                  // four sums: an addition waits for the one before
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
      const AdamEntry& e = t.e[find(t, chunk)];
      const long long at = (long long)(chunk - e.first) * kChunk;
      const int n = (int)min((long long)kChunk, e.n - at);
      if (e.bf16) squares(static_cast<const __nv_bfloat16*>(e.g) + at, n, e.vec, q);
      else squares(static_cast<const float*>(e.g) + at, n, e.vec, q);
    }
    double s = (q[0] + q[1]) + (q[2] + q[3]);
    s = block_sum(s, sm);
    if (threadIdx.x == 0) {
      a.parts[a.part0 + blockIdx.x] = s;
      __threadfence();
      final = atomicAdd(&a.ctl->ticket, 1u) == (unsigned)a.all_parts - 1u;
    }
    __syncthreads();
    if (!final) return;
    __threadfence();
    s = 0.0;
    for (int i = threadIdx.x; i < a.all_parts; i += kAdamThreads) s += __ldcg(a.parts + i);
    total = block_sum(s, sm);
  }
  // the last CTA, or the only one
  if (threadIdx.x == 0) {
    AdamControl& c = *a.ctl;
    bool ok = !a.loss || isfinite(*a.loss);
    float coef = 1.f;
    if (a.norm) {
      const float n = (float)sqrt(total), ema = c.ema;
      ok = ok && isfinite(n) && (a.spike <= 0.f || ema <= 0.f || n < a.spike * ema);
      if (a.clip > 0.f && n > a.clip) coef = __fdiv_rn(a.clip, n);      // clip may be infinite
      if (ok) c.ema = ema > 0.f ? __fadd_rn(__fmul_rn(0.98f, ema), __fmul_rn(0.02f, n)) : n;
      c.norm = n;
      c.ticket = 0;
    }
    c.ok = ok ? 1.f : 0.f;
    c.coef = coef;
    go = ok;
  }
  __syncthreads();
  if (a.alone && go) count_up(t);
}

// The factors of one of several tables.
template <int N>
__global__ void __launch_bounds__(kAdamThreads) adamw_prepare_kernel(const __grid_constant__ AdamTable<N> t,
                                                                     const __grid_constant__ AdamParams a) {
  pdl_enter();
  if (a.ctl->ok == 0.f) return;
  factors(t, a);
  __syncthreads();
  count_up(t);
}

// Two fp32 values in a register pair: one instruction multiplies both, each rounded to nearest.  Sums of two products
// are scalar: a packed sum came out joined with its product, rounded once.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ void apart(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two add(Two a, Two b) {
  float x[2], y[2];
  apart(a, x[0], x[1]);
  apart(b, y[0], y[1]);
  return two(__fadd_rn(x[0], y[0]), __fadd_rn(x[1], y[1]));
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

struct Steps {                          // a tensor's factors and the step's, twice each
  Two size, root, decay, coef, b1, g1, b2, g2, eps;
};
__device__ __forceinline__ Steps steps_of(const Factors& f, const AdamParams& a, float coef) {
  return {both(-f.size), both(f.root), both(f.decay), both(coef), both(a.fb1), both(a.gb1), both(a.fb2), both(a.gb2), both(a.eps)};
}
// Two values' moments, every operation rounded by itself.
__device__ __forceinline__ void moments(Two g, Two& m, Two& v, const Steps& s) {
  g = mul(g, s.coef);
  m = add(mul(s.b1, m), mul(s.g1, g));
  v = add(mul(s.b2, v), mul(s.g2, mul(g, g)));
}
// Their step from m and the roots of v.  The approximate root and reciprocal and the products leave the step within some 4 ulp
// of itself, 2^-21: two roundings more than an exact division would, whatever the size of p.
__device__ __forceinline__ Two stepped(Two p, Two m, Two r, const Steps& s) {
  float a, b;
  apart(fma(r, s.root, s.eps), a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return fma(p, s.decay, mul(s.size, mul(m, two(a, b))));
}
__device__ __forceinline__ float root_near(float v) {  // within an ulp
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Loads of memory that the kernel also writes.
__device__ __forceinline__ void own4(const float* p, float v[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void own4(const __nv_bfloat16* p, float v[4]) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
  v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
}
__device__ __forceinline__ float own1(const float* p) { return *p; }
__device__ __forceinline__ float own1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <class T>
__device__ __forceinline__ void load4(const T* p, float v[4], bool vec, int n) {
  if (vec) {
    own4(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? own1(p + j) : 0.f;
  }
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <class T>
__device__ __forceinline__ void store4(T* p, const float v[4], bool vec, int n) {
  if (vec) {
    st4(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) store1(p + j, v[j]);
  }
}
__device__ __forceinline__ uint32_t codes4(const uint8_t* p, bool vec, int n) {
  if (vec) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) c |= (uint32_t)p[j] << (8 * j);
  return c;
}
__device__ __forceinline__ void codes4(uint8_t* p, uint32_t c, bool vec, int n) {
  if (vec) {
    *reinterpret_cast<uint32_t*>(p) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = (uint8_t)(c >> (8 * j));
  }
}

// The values of four codes, in pairs.
__device__ __forceinline__ void decode_m(uint32_t c, Two scale, Two v[2]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * j)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[j] = mul(two(f.x, f.y), scale);
  }
}
__device__ __forceinline__ void decode_v(uint32_t c, Two scale, Two v[2]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    // a code's bits are a float's exponent and mantissa, 2^112 too small
    const uint32_t lo = (j ? c << 3 : c << 19) & 0x07f80000u, hi = (j ? c >> 5 : c << 11) & 0x07f80000u;
    const Two r = mul(mul(two(__uint_as_float(lo), __uint_as_float(hi)), both(0x1p112f)), scale);
    v[j] = mul(r, r);
  }
}
// The scale of a warp's block from its lanes' largest magnitude, as bits (so that a NaN is the largest), and what values
// are multiplied by (0: all are stored as zero).
__device__ __forceinline__ float scale_of(uint32_t largest, float inverse_top, float& up) {
  const float s = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, largest)), inverse_top);
  up = s >= kNormal ? __frcp_rn(s) : 0.f;
  return s;
}
__device__ __forceinline__ uint32_t encode_m(const Two v[2], Two up) {
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float2 f;                           // at most 448 and an ulp
    apart(mul(v[j], up), f.x, f.y);
    c |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (16 * j);
  }
  return c;
}
__device__ __forceinline__ uint32_t encode_r(const Two r[2], Two up) {
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x[2], w[2];                   // x: at most 1.9375 and an ulp
    apart(mul(r[j / 2], up), x[0], x[1]);
    apart(r[j / 2], w[0], w[1]);
    const float y = x[j & 1];
    const uint32_t u = __float_as_uint(y);
    // to nearest, ties to even: at a normal number's fourth bit, or below 2^-14 to a multiple of 2^-18 (in the low bits
    // of a sum with 1.5 x 2^23)
    uint32_t k = y >= 0x1p-14f ? ((u + 0x3ffffu + ((u >> 19) & 1u)) >> 19) - (112u << 4)
                               : __float_as_uint(__fmaf_rn(y, 0x1p18f, 12582912.f)) & 31u;
    k = max(k, min(__float_as_uint(w[j & 1]), 1u));   // a root above zero is at least code 1
    c |= (k & 255u) << (8 * j);
  }
  return c;
}

// 4 values of a thread, 8 bits: 8 of a lane, a warp to a block.  WHOLE: a full chunk, read 4 values at a time.
template <class T, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void chunk_update(const AdamEntry& e, const Steps& st, long long at, int n) {
  T* p = static_cast<T*>(e.p) + at;
  const T* g = static_cast<const T*>(e.g) + at;
  auto pairs = [](const float v[4], Two q[2]) { q[0] = two(v[0], v[1]); q[1] = two(v[2], v[3]); };
  auto singles = [](const Two q[2], float v[4]) { apart(q[0], v[0], v[1]); apart(q[1], v[2], v[3]); };
  if constexpr (!EIGHT) {
    float* m = static_cast<float*>(e.m) + at;
    float* v = static_cast<float*>(e.v) + at;
    for (int i0 = threadIdx.x * 4; i0 < n; i0 += kAdamThreads * 8) {  // two at a time: their loads come first
      float x[2][4], y[2][4], mm[2][4], vv[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = i0 + h * kAdamThreads * 4;
        const bool vec = WHOLE || (e.vec && i + 4 <= n);
        load4(p + i, x[h], vec, n - i);
        load4(g + i, y[h], vec, n - i);
        load4(m + i, mm[h], vec, n - i);
        load4(v + i, vv[h], vec, n - i);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = i0 + h * kAdamThreads * 4;
        const bool vec = WHOLE || (e.vec && i + 4 <= n);
        Two xs[2], gs[2], ms[2], vs[2];
        pairs(x[h], xs);
        pairs(y[h], gs);
        pairs(mm[h], ms);
        pairs(vv[h], vs);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          moments(gs[j], ms[j], vs[j], st);
          float a, b;
          apart(vs[j], a, b);
          xs[j] = stepped(xs[j], ms[j], two(root_near(a), root_near(b)), st);
        }
        singles(xs, x[h]);
        singles(ms, mm[h]);
        singles(vs, vv[h]);
        store4(p + i, x[h], vec, n - i);
        store4(m + i, mm[h], vec, n - i);
        store4(v + i, vv[h], vec, n - i);
      }
    }
  } else {
    uint8_t* m = static_cast<uint8_t*>(e.m) + at;
    uint8_t* v = static_cast<uint8_t*>(e.v) + at;
    float* m_scale = e.ms + at / kBlock;
    float* v_scale = e.vs + at / kBlock;
    const int lane = threadIdx.x & 31;
    float nx[2][4], ny[2][4], nms, nvs;
    uint32_t ncm[2], ncv[2];
    auto load = [&](int blk) {
      nms = m_scale[blk];
      nvs = v_scale[blk];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = blk * kBlock + h * 128 + lane * 4;
        const bool vec = WHOLE || (e.vec && n - i >= 4);
        load4(p + i, nx[h], vec, n - i);
        load4(g + i, ny[h], vec, n - i);
        ncm[h] = codes4(m + i, vec, n - i);
        ncv[h] = codes4(v + i, vec, n - i);
      }
    };
    if (WHOLE) load(threadIdx.x >> 5);
    for (int blk = threadIdx.x >> 5; blk * kBlock < n; blk += kAdamThreads / 32) {
      if (!WHOLE) load(blk);
      const float ms = nms, vs = nvs;
      float x[2][4], y[2][4];
      Two mm[2][2], r[2][2];
      uint32_t cm[2], cv[2], top_m = 0, top_r = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cm[h] = ncm[h];
        cv[h] = ncv[h];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[h][j] = nx[h][j];
          y[h][j] = ny[h][j];
        }
      }
      if (WHOLE && blk + kAdamThreads / 32 < kChunk / kBlock) load(blk + kAdamThreads / 32);  // before this block's work
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = n - (blk * kBlock + h * 128 + lane * 4);
        Two xs[2], gs[2], vv[2];
        pairs(x[h], xs);
        pairs(y[h], gs);
        decode_m(cm[h], both(ms), mm[h]);
        decode_v(cv[h], both(vs), vv);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          moments(gs[j], mm[h][j], vv[j], st);
          float a, b, c, d;
          apart(mm[h][j], a, b);
          apart(vv[j], c, d);
          if (!WHOLE) {                 // past the tensor's end
            if (2 * j >= left) a = c = 0.f;
            if (2 * j + 1 >= left) b = d = 0.f;
            mm[h][j] = two(a, b);
          }
          c = __fsqrt_rn(c);
          d = __fsqrt_rn(d);
          r[h][j] = two(c, d);
          xs[j] = stepped(xs[j], mm[h][j], r[h][j], st);
          top_m = max(top_m, max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
          top_r = max(top_r, max(__float_as_uint(c) & 0x7fffffffu, __float_as_uint(d) & 0x7fffffffu));
        }
        singles(xs, x[h]);
      }
      float up_m, up_r;
      const float new_ms = scale_of(top_m, 1.f / 448.f, up_m), new_vs = scale_of(top_r, 1.f / 1.9375f, up_r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = blk * kBlock + h * 128 + lane * 4;
        const bool vec = WHOLE || (e.vec && n - i >= 4);
        store4(p + i, x[h], vec, n - i);
        codes4(m + i, encode_m(mm[h], both(up_m)), vec, n - i);
        codes4(v + i, encode_r(r[h], both(up_r)), vec, n - i);
      }
      if (lane == 0) {
        m_scale[blk] = new_ms;
        v_scale[blk] = new_vs;
      }
    }
  }
}

template <int N, bool EIGHT>
__global__ void __launch_bounds__(kAdamThreads, EIGHT ? 3 : 4) adamw_update_kernel(const __grid_constant__ AdamTable<N> t,
                                                                    const __grid_constant__ AdamParams a) {
  pdl_enter();
  if (__ldcg(&a.ctl->ok) == 0.f) return;
  const float coef = __ldcg(&a.ctl->coef);
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int i = find(t, chunk);
    const AdamEntry& e = t.e[i];
    const Factors& from = a.factors[a.tensor0 + i];
    const Factors f = {__ldcg(&from.size), __ldcg(&from.root), __ldcg(&from.decay)};
    const long long at = (long long)(chunk - e.first) * kChunk;
    const int n = (int)min((long long)kChunk, e.n - at);
    const bool whole = e.vec && n == kChunk;
    const Steps s = steps_of(f, a, coef);
    if (e.bf16)
      whole ? chunk_update<__nv_bfloat16, EIGHT, true>(e, s, at, kChunk) : chunk_update<__nv_bfloat16, EIGHT, false>(e, s, at, n);
    else
      whole ? chunk_update<float, EIGHT, true>(e, s, at, kChunk) : chunk_update<float, EIGHT, false>(e, s, at, n);
  }
}

// What 8-bit moments stand for: m and v in fp32, to where the entry's p and g point.
template <int N>
__global__ void __launch_bounds__(kAdamThreads) adamw_moments_kernel(const __grid_constant__ AdamTable<N> t) {
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const AdamEntry& e = t.e[find(t, chunk)];
    const long long at = (long long)(chunk - e.first) * kChunk;
    const int n = (int)min((long long)kChunk, e.n - at);
    const uint8_t* m = static_cast<const uint8_t*>(e.m) + at;
    const uint8_t* v = static_cast<const uint8_t*>(e.v) + at;
    float* om = static_cast<float*>(e.p) + at;
    float* ov = static_cast<float*>(const_cast<void*>(e.g)) + at;
    const int lane = threadIdx.x & 31;
#pragma unroll 2
    for (int blk = threadIdx.x >> 5; blk * kBlock < n; blk += kAdamThreads / 32) {
      const float ms = e.ms[at / kBlock + blk], vs = e.vs[at / kBlock + blk];
      uint32_t cm[2], cv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = blk * kBlock + h * 128 + lane * 4;
        cm[h] = codes4(m + i, e.vec && n - i >= 4, n - i);
        cv[h] = codes4(v + i, e.vec && n - i >= 4, n - i);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = blk * kBlock + h * 128 + lane * 4;
        float x[4];
        Two q[2];
        decode_m(cm[h], both(ms), q);
        apart(q[0], x[0], x[1]);
        apart(q[1], x[2], x[3]);
        store4(om + i, x, e.vec && n - i >= 4, n - i);
        decode_v(cv[h], both(vs), q);
        apart(q[0], x[0], x[1]);
        apart(q[1], x[2], x[3]);
        store4(ov + i, x, e.vec && n - i >= 4, n - i);
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------
constexpr int kFew = 32, kMany = 320;  // tensors of a table: 3 and 31 KB of parameters

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

gdn2_status check_adamw(const gdn2_adamw_desc* d, const gdn2_adamw_tensor* ts, int32_t n) {
  if (!d || n < 0 || (n && !ts) || (d->state_bits != 32 && d->state_bits != 8)) return GDN2_ERR_INVALID_ARGUMENT;
  if (!(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1 && d->eps >= 0 && d->clip >= 0 && d->spike >= 0))
    return GDN2_ERR_INVALID_ARGUMENT;
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    const gdn2_adamw_tensor& t = ts[i];
    if (t.n < 0 || (t.dtype != GDN2_F32 && t.dtype != GDN2_BF16)) return GDN2_ERR_INVALID_ARGUMENT;
    if (t.n > 1ll << 42) return GDN2_ERR_UNSUPPORTED;
    if (!t.n) continue;
    const size_t el = t.dtype == GDN2_BF16 ? 2 : 4, st = d->state_bits == 8 ? 1 : 4;
    if (!t.p || !t.g || !t.m || !t.v || !aligned(t.p, el) || !aligned(t.g, el) || !aligned(t.m, st) || !aligned(t.v, st))
      return GDN2_ERR_INVALID_ARGUMENT;
    if (st == 1 && (!t.m_scale || !t.v_scale || !aligned(t.m_scale, 4) || !aligned(t.v_scale, 4)))
      return GDN2_ERR_INVALID_ARGUMENT;
    chunks += (t.n + kChunk - 1) / kChunk;
  }
  return chunks < 1ll << 30 ? GDN2_OK : GDN2_ERR_UNSUPPORTED;
}

// Fills a table from ts[i..) and returns the next index.
template <int N>
int fill(AdamTable<N>& t, const gdn2_adamw_desc* d, const gdn2_adamw_tensor* ts, int i, int n) {
  t.count = t.chunks = 0;
  const size_t st = d->state_bits == 8 ? 4 : 16;
  for (; i < n && t.count < N; ++i) {
    const gdn2_adamw_tensor& s = ts[i];
    if (!s.n) continue;
    const size_t el = s.dtype == GDN2_BF16 ? 8 : 16;
    AdamEntry& e = t.e[t.count++];
    e.p = s.p; e.g = s.g; e.m = s.m; e.v = s.v; e.ms = s.m_scale; e.vs = s.v_scale;
    e.step = s.step; e.lr_at = s.lr_at; e.lr = s.lr; e.wd = s.weight_decay; e.n = s.n;
    e.first = t.chunks;
    e.bf16 = s.dtype == GDN2_BF16;
    e.vec = aligned(s.p, el) && aligned(s.g, el) && aligned(s.m, st) && aligned(s.v, st);
    t.chunks += (int)((s.n + kChunk - 1) / kChunk);
  }
  return i;
}

constexpr int kMostCtas = 148 * 5;          // as many as are at work at a time
int norm_grid(int chunks) { return chunks < kMostCtas ? chunks : kMostCtas; }
struct AdamTotal {
  int tensors, parts;                   // parts: CTAs of the norm's launches
};
// Tables have `most` tensors.
AdamTotal totals(const gdn2_adamw_tensor* ts, int n, int most) {
  AdamTotal r{0, 0};
  int chunks = 0, in = 0;
  for (int i = 0; i < n; ++i) {
    if (!ts[i].n) continue;
    if (in == most) {
      r.parts += norm_grid(chunks);
      chunks = in = 0;
    }
    ++in;
    ++r.tensors;
    chunks += (int)((ts[i].n + kChunk - 1) / kChunk);
  }
  r.parts += norm_grid(chunks);
  return r;
}
size_t parts_bytes(int parts) { return ((size_t)parts * sizeof(double) + 255) / 256 * 256; }

template <int N>
cudaError_t run_adamw(const gdn2_adamw_desc* d, const gdn2_adamw_tensor* ts, int n, AdamParams a, cudaStream_t st) {
  static thread_local AdamTable<N> t;  // 31 KB: not on the stack
  cudaError_t e = cudaSuccess;
  const AdamTotal all = totals(ts, n, N);
  a.alone = all.tensors <= N;
  a.all_parts = all.parts;
  a.part0 = a.tensor0 = 0;
  if (a.norm || a.alone) {
    for (int i = 0; i < n && e == cudaSuccess;) {
      i = fill(t, d, ts, i, n);
      if (!t.count) break;
      const int grid = a.norm ? norm_grid(t.chunks) : 1;
      e = launch_pdl(adamw_norm_kernel<N>, grid, kAdamThreads, 0, st, t, a);
      a.part0 += grid;
    }
  }
  if (!a.alone) {
    if (!a.norm && e == cudaSuccess) {  // the guard alone, over no tensors
      t.count = t.chunks = 0;
      e = launch_pdl(adamw_norm_kernel<N>, 1, kAdamThreads, 0, st, t, a);
    }
    for (int i = 0; i < n && e == cudaSuccess;) {
      i = fill(t, d, ts, i, n);
      if (!t.count) break;
      e = launch_pdl(adamw_prepare_kernel<N>, 1, kAdamThreads, 0, st, t, a);
      a.tensor0 += t.count;
    }
    a.tensor0 = 0;
  }
  for (int i = 0; i < n && e == cudaSuccess;) {
    i = fill(t, d, ts, i, n);
    if (!t.count) break;
    // codes: as many CTAs as are at work at a time, each walks its chunks (8 bits, 39 M fp32 weights: 125 us; 132 with
    // 1184 CTAs, 146 with one for each chunk); 32 bits move more bytes than they compute and are better off with the
    // scheduler's order (39 M weights: 161, not 174 us)
    const unsigned grid = (unsigned)(d->state_bits == 8 && t.chunks > 148 * 3 ? 148 * 3 : t.chunks);
    e = d->state_bits == 8 ? launch_pdl(adamw_update_kernel<N, true>, grid, kAdamThreads, 0, st, t, a)
                           : launch_pdl(adamw_update_kernel<N, false>, grid, kAdamThreads, 0, st, t, a);
    a.tensor0 += t.count;
  }
  return e;
}

template <int N>
cudaError_t run_moments(const gdn2_adamw_desc* d, const gdn2_adamw_tensor* ts, int n, cudaStream_t st) {
  static thread_local AdamTable<N> t;
  for (int i = 0; i < n;) {
    i = fill(t, d, ts, i, n);
    if (!t.count) break;
    adamw_moments_kernel<N><<<(unsigned)t.chunks, kAdamThreads, 0, st>>>(t);
  }
  return cudaGetLastError();
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_adamw_workspace_bytes(const gdn2_adamw_desc* d, const gdn2_adamw_tensor* tensors, int32_t n) {
  using namespace gdn2;
  if (check_adamw(d, tensors, n) != GDN2_OK) return 0;
  const AdamTotal all = totals(tensors, n, kMany);
  return all.tensors ? parts_bytes(all.parts) + all.tensors * sizeof(Factors) : 0;
}

extern "C" gdn2_status gdn2_adamw_step(const gdn2_adamw_desc* d, const gdn2_adamw_tensor* tensors, int32_t n,
                                       const float* loss, void* control, void* workspace, void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_adamw(d, tensors, n);
  if (s != GDN2_OK) return s;
  const AdamTotal all = totals(tensors, n, kMany);
  if (!all.tensors) return GDN2_OK;
  for (int i = 0; i < n; ++i)
    if (tensors[i].n && (!tensors[i].step || !aligned(tensors[i].step, 4))) return GDN2_ERR_INVALID_ARGUMENT;
  if (!control || !aligned(control, 4) || !workspace || !aligned(workspace, 256)) return GDN2_ERR_INVALID_ARGUMENT;
  AdamParams a{};
  a.ctl = static_cast<AdamControl*>(control);
  a.parts = static_cast<double*>(workspace);
  a.factors = reinterpret_cast<Factors*>(static_cast<uint8_t*>(workspace) + parts_bytes(all.parts));
  a.loss = loss;
  a.log2_b1 = log2(d->beta1); a.log2_b2 = log2(d->beta2);
  a.fb1 = (float)d->beta1; a.gb1 = (float)(1.0 - d->beta1);
  a.fb2 = (float)d->beta2; a.gb2 = (float)(1.0 - d->beta2);
  a.eps = (float)d->eps;
  // above zero they stay so in fp32
  a.clip = d->clip > 0 ? fmaxf((float)d->clip, kNormal) : 0.f;
  a.spike = d->spike > 0 ? fmaxf((float)d->spike, kNormal) : 0.f;
  a.norm = d->clip > 0 || d->spike > 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = all.tensors <= kFew ? run_adamw<kFew>(d, tensors, n, a, st) : run_adamw<kMany>(d, tensors, n, a, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}

extern "C" gdn2_status gdn2_adamw_moments(const gdn2_adamw_tensor* tensors, int32_t n, void* stream) {
  using namespace gdn2;
  gdn2_adamw_desc d{};
  d.state_bits = 8;
  const gdn2_status s = check_adamw(&d, tensors, n);
  if (s != GDN2_OK) return s;
  for (int i = 0; i < n; ++i)
    if (tensors[i].dtype != GDN2_F32) return GDN2_ERR_INVALID_ARGUMENT;
  const AdamTotal all = totals(tensors, n, kMany);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = all.tensors <= kFew ? run_moments<kFew>(&d, tensors, n, st) : run_moments<kMany>(&d, tensors, n, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
