// Products of a few rows with a 4-bit weight (sm_100a):
//   y[m, n] = act( sum_G s[G, n] sum_{k in G} Q[k, n] x[m, k] + bias[n] ) + residual[m, n]
// Q holds integers in [-8, 7], s one scale (bf16) per group of 32, 64 or 128 rows of a column.
//
// The weight is read once, at half a byte per element, and that bounds the product for few rows.
// Widening and multiplying on the CUDA cores would need more issue slots per byte than the HBM
// rate leaves, so the products go to the warp-level tensor instruction (m16n8k16, bf16 operands,
// fp32 accumulators) with the weight as the 16-row operand and eight rows of x as its columns:
// integers in [-8, 7] are exact in bf16, products with bf16 x are exact in fp32, and the scale is
// applied in fp32 to each group's sum.  fp32 x is split into three bf16 terms (24 bits), one
// instruction each.
//
// Packed weight (W4Weight in w4.py): tiles of 16 columns x 64 rows, 512 bytes each, the tiles of a
// column block contiguous along k.  A lane (g = lane / 4, t = lane % 4) owns 16 bytes of a tile:
// word s (k-step s of 4) has eight nibbles Q + 8; with k = 32 (s / 2) + 8 t + 4 (s % 2) + j,
// nibble r + 4 (j % 2), r = 2 (j / 2) + c, is column g + 8 c.  The sum over k may run in any
// order: this one puts the x values a lane needs for two k-steps next to one another.
#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

struct W4Params {
  const void* x;
  const uint4* w;
  const __nv_bfloat16* scales;  // (column blocks, groups, 16)
  const float* bias;
  const void* res;
  void* y;
  long long xs, rs, ys;  // row strides in elements
  int M, K, N, KB, groups, gshift;  // gshift: log2 of the group
  int gelu;
};

__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight nibbles -> four bf16 pairs.  0x4300 is 128, whose last mantissa bit is worth 1: 128 + Q + 8
// by an OR, then 136 is subtracted; both are exact.
__device__ __forceinline__ void widen(uint32_t w, uint32_t a[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    uint32_t v = ((w >> (4 * r)) & 0x000f000fu) | 0x43004300u;
    const uint32_t off = 0x43084308u;
    __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
    a[r] = *reinterpret_cast<uint32_t*>(&d);
  }
}

__device__ __forceinline__ float gelu_tanh(float y) {
  return 0.5f * y * (1.f + tanhf(0.7978845608028654f * (y + 0.044715f * y * y * y)));
}

// Eight neighbouring values of row m from column k on (zeros outside) as kTerms bf16 terms.
template <class T, int kTerms>
__device__ __forceinline__ void load_x(const W4Params& p, int m, int k, bool vec, uint32_t f[kTerms][4]) {
  float v[8];
  const T* src = static_cast<const T*>(p.x) + (long long)m * p.xs + k;
  if (m < p.M && vec && k + 8 <= p.K) {
    float lo[4], hi[4];
    ld4(src, lo);
    ld4(src + 4, hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m < p.M && k + i < p.K ? ld1(src + i) : 0.f;
  }
#pragma unroll
  for (int t = 0; t < kTerms; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      f[t][i] = *reinterpret_cast<const uint32_t*>(&h);
      if (t + 1 < kTerms) {  // the term's remainder (an infinity leaves none)
        const float2 back = __bfloat1622float2(h);
        v[2 * i] = isinf(back.x) ? 0.f : v[2 * i] - back.x;
        v[2 * i + 1] = isinf(back.y) ? 0.f : v[2 * i + 1] - back.y;
      }
    }
}

constexpr int kW4Warps = 8;

// A CTA: kNT blocks of 16 columns x 8 kMB rows; its warps take the 64-row tiles in turn.
template <class T, int kTerms, int kNT, int kMB>
__global__ void __launch_bounds__(kW4Warps * 32) w4_kernel(W4Params p, bool vec) {
  __shared__ float part[kW4Warps][kNT * 16][kMB * 8 + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int nb0 = blockIdx.x * kNT, NB = (p.N + 15) >> 4;
  const int m0 = blockIdx.y * kMB * 8;
  float sum[kNT][kMB][4];
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int j = 0; j < kMB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[i][j][c] = 0.f;
  for (int kb = warp; kb < p.KB; kb += kW4Warps) {
    uint4 w[kNT];
#pragma unroll
    for (int i = 0; i < kNT; ++i)
      w[i] = nb0 + i < NB ? __ldg(p.w + ((size_t)(nb0 + i) * p.KB + kb) * 32 + lane)
                          : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t f[kMB][kTerms][4];
#pragma unroll
      for (int j = 0; j < kMB; ++j)
        load_x<T, kTerms>(p, m0 + j * 8 + g, kb * 64 + half * 32 + t * 8, vec, f[j]);
      const int grp = min((kb * 64 + half * 32) >> p.gshift, p.groups - 1);
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        uint32_t a0[4], a1[4];
        widen(half ? w[i].z : w[i].x, a0);
        widen(half ? w[i].w : w[i].y, a1);
        const __nv_bfloat16* sc = p.scales + ((size_t)min(nb0 + i, NB - 1) * p.groups + grp) * 16;
        const float s0 = __bfloat162float(sc[g]), s1 = __bfloat162float(sc[g + 8]);
#pragma unroll
        for (int j = 0; j < kMB; ++j) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = kTerms - 1; e >= 0; --e) {
            mma16816(acc, a0, f[j][e][0], f[j][e][1]);
            mma16816(acc, a1, f[j][e][2], f[j][e][3]);
          }
          sum[i][j][0] = fmaf(s0, acc[0], sum[i][j][0]);
          sum[i][j][1] = fmaf(s0, acc[1], sum[i][j][1]);
          sum[i][j][2] = fmaf(s1, acc[2], sum[i][j][2]);
          sum[i][j][3] = fmaf(s1, acc[3], sum[i][j][3]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int j = 0; j < kMB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        part[warp][i * 16 + g + (c >> 1) * 8][j * 8 + 2 * t + (c & 1)] = sum[i][j][c];
  __syncthreads();
  for (int e = tid; e < kNT * 16 * kMB * 8; e += kW4Warps * 32) {
    const int n = e % (kNT * 16), m = e / (kNT * 16);
    const int col = nb0 * 16 + n, row = m0 + m;
    if (col >= p.N || row >= p.M) continue;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < kW4Warps; ++i) y += part[i][n][m];
    if (p.bias) y += p.bias[col];
    if (p.gelu) y = gelu_tanh(y);
    if (p.res) y += ld1(static_cast<const T*>(p.res) + (long long)row * p.rs + col);
    if constexpr (sizeof(T) == 2) static_cast<__nv_bfloat16*>(p.y)[(long long)row * p.ys + col] = __float2bfloat16(y);
    else static_cast<float*>(p.y)[(long long)row * p.ys + col] = y;
  }
}

template <class T, int kTerms>
void launch(const W4Params& p, bool vec, cudaStream_t st) {
  const int NB = (p.N + 15) / 16;
  if (p.M <= 8)
    w4_kernel<T, kTerms, 2, 1><<<dim3((NB + 1) / 2, 1), kW4Warps * 32, 0, st>>>(p, vec);
  else
    w4_kernel<T, kTerms, 2, 2><<<dim3((NB + 1) / 2, (p.M + 15) / 16), kW4Warps * 32, 0, st>>>(p, vec);
}

}  // namespace
}  // namespace gdn2

extern "C" gdn2_status gdn2_w4_linear(const gdn2_w4_desc* d, const void* x, const void* packed, const void* scales,
                                      const float* bias, const void* residual, void* y, void* stream) {
  using namespace gdn2;
  if (!d || d->M <= 0 || d->K <= 0 || d->N <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->group != 32 && d->group != 64 && d->group != 128) return GDN2_ERR_UNSUPPORTED;
  if (d->act != GDN2_ACT_NONE && d->act != GDN2_ACT_GELU_TANH) return GDN2_ERR_INVALID_ARGUMENT;
  if (!x || !packed || !scales || !y || (reinterpret_cast<uintptr_t>(packed) & 15u)) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->x_stride < 0 || d->y_stride < d->N || (residual && d->res_stride < 0)) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->M > 65535 * 16) return GDN2_ERR_UNSUPPORTED;
  const int el = d->dtype == GDN2_BF16 ? 2 : 4;
  W4Params p{};
  p.x = x;
  p.w = static_cast<const uint4*>(packed);
  p.scales = static_cast<const __nv_bfloat16*>(scales);
  p.bias = bias; p.res = residual; p.y = y;
  p.xs = d->x_stride; p.rs = d->res_stride; p.ys = d->y_stride;
  p.M = d->M; p.K = d->K; p.N = d->N;
  p.KB = (d->K + 63) / 64;
  p.groups = (d->K + d->group - 1) / d->group;
  p.gshift = d->group == 32 ? 5 : d->group == 64 ? 6 : 7;
  p.gelu = d->act == GDN2_ACT_GELU_TANH;
  // rows whose every eighth value starts on 16 bytes are loaded as vectors
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (d->x_stride * el) % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (el == 2) launch<__nv_bfloat16, 1>(p, vec, st);
  else launch<float, 3>(p, vec, st);
  return cudaGetLastError() == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
