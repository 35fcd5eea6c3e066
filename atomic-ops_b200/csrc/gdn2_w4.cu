// Products of a few rows with a 4-bit weight (sm_100a):
//   y[m, n] = act( sum_G s[G, n] sum_{k in G} Q[k, n] x[m, k] + bias[n] ) + residual[m, n]
// Q holds integers in [-8, 7], s one scale (bf16) per group of 32, 64 or 128 rows of a column.
//
// The weight is read once, at half a byte per element, and that bounds the product for few rows;
// what competes with it is the issue slots that widening takes.  Multiplying on the CUDA cores would
// need one more slot per weight and row, so the products go to the warp-level tensor instruction
// (m16n8k16, bf16 operands, fp32 accumulators) with the weight as the 16-row operand and eight rows
// of x as its columns: integers in [-8, 7] are exact in bf16, products with bf16 x are exact in fp32,
// and the scale is applied in fp32 to each group's sum.  fp32 x is cut into three bf16 terms of 8
// bits (exact), one instruction each.
//
// Packed weight (W4Weight in w4.py): tiles of 16 columns x 64 rows, 512 bytes each; the two tiles of
// 32 columns lie next to one another, then the next 64 rows.  A lane (g = lane / 4, t = lane % 4)
// owns 16 bytes of a tile: word s (k-step s of 4) has eight nibbles Q + 8; with
// k = 32 (s / 2) + 8 t + 4 (s % 2) + j, nibble r + 4 (j % 2), r = 2 (j / 2) + c, is column g + 8 c.
// The sum over k may run in any order: this one puts the x values that a lane needs for two k-steps
// next to one another, so that rows of x on 16 bytes are read as they are.
#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

constexpr int kW4Warps = 8;
constexpr int kSmCount = 148;  // of a B200

struct W4Params {
  const void* x;
  const uint4* xp;        // x as terms in the order in which the lanes read them, or null
  const uint4* w;
  const uint8_t* scales;
  const float* bias;
  const void* res;
  void* y;
  long long xs, rs, ys;  // row strides in elements
  int M, K, N, NB, gelu;  // NB: batches of 128 rows of the weight
};

__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight nibbles -> four bf16 pairs.  0x4300 is 128, whose last mantissa bit is worth 1: 136 + Q by an
// OR; subtracting 136 is exact.
__device__ __forceinline__ void widen(uint32_t w, uint32_t a[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    uint32_t v = ((w >> (4 * r)) & 0x000f000fu) | 0x43004300u;
    const uint32_t off = 0x43084308u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
    a[r] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

__device__ __forceinline__ float gelu_tanh(float y) {
  return 0.5f * y * (1.f + tanhf(0.7978845608028654f * (y + 0.044715f * y * y * y)));
}

// Eight fp32 as three bf16 terms of 8 bits each, the upper half of what is left: exact.
__device__ __forceinline__ void cut(float v[8], uint32_t f[3][4]) {
#pragma unroll
  for (int t = 0; t < 3; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[t][i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
    if (t < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float rest = v[i] - __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u);
        v[i] = rest == rest ? rest : 0.f;  // an infinity or a NaN is in the first term alone
      }
    }
  }
}

// Terms of x in the lanes' order: [row block of 8 kMB][128-row batch][4 x 32][8 rows][term][lane].
// For rows that are not on 16 bytes, and for fp32 where many column blocks would repeat the cut.
template <class T>
__global__ void __launch_bounds__(256) w4_terms_kernel(W4Params p, uint4* out, int mb) {
  constexpr int kTerms = sizeof(T) == 2 ? 1 : 3;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);  // ((block, batch, quarter), j)
  const int j = (int)(unit % mb);
  const long long q = unit / mb;
  const long long nq = (long long)p.NB * 4;
  const int m = (int)(q / nq) * mb * 8 + j * 8 + g, k = (int)(q % nq) * 32 + t * 8;
  if ((q / nq) * mb * 8 < p.M) {
    const T* src = static_cast<const T*>(p.x) + (long long)m * p.xs + k;
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m < p.M && k + i < p.K ? src[i] : T(0.f);
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)__bfloat16_as_ushort(v[2 * i]) | (uint32_t)__bfloat16_as_ushort(v[2 * i + 1]) << 16;
      out[unit * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      uint32_t f[3][4];
      cut(v, f);
#pragma unroll
      for (int e = 0; e < kTerms; ++e)
        out[(unit * kTerms + e) * 32 + lane] = make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]);
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// One 32-row quarter of a batch for kMB blocks of eight rows of x.
template <class T, int kTerms, int kMB, bool kPacked>
__device__ __forceinline__ void load_quarter(const W4Params& p, const T* const xsrc[kMB], const uint4* xp, int k,
                                             uint32_t f[kMB][kTerms][4]) {
#pragma unroll
  for (int j = 0; j < kMB; ++j) {
    if constexpr (kPacked) {
#pragma unroll
      for (int e = 0; e < kTerms; ++e) {
        const uint4 v = xp[(j * kTerms + e) * 32];  // not __ldg: the grid before may still write it when this one starts
        f[j][e][0] = v.x; f[j][e][1] = v.y; f[j][e][2] = v.z; f[j][e][3] = v.w;
      }
    } else if constexpr (sizeof(T) == 2) {
      const uint4 v = k < p.K ? __ldg(reinterpret_cast<const uint4*>(xsrc[j])) : make_uint4(0u, 0u, 0u, 0u);
      f[j][0][0] = v.x; f[j][0][1] = v.y; f[j][0][2] = v.z; f[j][0][3] = v.w;
    } else {
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 a = k < p.K ? __ldg(reinterpret_cast<const float4*>(xsrc[j])) : z;
      const float4 b = k < p.K ? __ldg(reinterpret_cast<const float4*>(xsrc[j]) + 1) : z;
      float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      cut(v, f[j]);
    }
  }
}

// Two CTAs on an SM where the registers allow.
template <int kTerms, int kMB>
constexpr bool kTwoCtas = kMB == 1 || (kTerms == 1 && kMB == 2);

// A warp computes 32 columns for 8 kMB rows over its share of the batches of 128 rows; a CTA has kMB
// warps side by side (they share x through L1) and 8 / kMB that split the batches, and the CTAs of a
// cluster split them further.  kPer: scales of a column per batch.
//
// Bound, where there are many columns, by the waits for its loads (a batch ahead; it issues in half of the
// cycles), then by the slots that widening takes.  Measured (bf16): 4 x 8192 x 8192 11.8 us (2.9 TB/s of
// weight), 16 x 8192 x 8192 16.1 us, 32 x 5000 x 12345 35.4 us, 8 x 2048 x 512 3.7 us.  Widening takes 136 out
// of every value before the product: leaving it in and taking 136 sum x out of the group's sum costs the bits
// of every x that is far below the group's largest, and was no faster (12.2 us).
template <class T, int kTerms, int kMB, int kPer, bool kPacked>
__global__ void __launch_bounds__(kW4Warps * 32, kTwoCtas<kTerms, kMB> ? 2 : 1) w4_kernel(W4Params p) {
  constexpr int kWN = kMB, kWK = kW4Warps / kWN, kCols = kWN * 32, kRows = kMB * 8 + 1;
  __shared__ float part[kW4Warps * 32 * kRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wk = warp / kWN, wn = warp % kWN;
  const int g = lane >> 2, t = lane & 3;
  const int ksplit = gridDim.y, m0 = blockIdx.z * kMB * 8;
  // column blocks past the weight's are read as its last one and not stored
  const int cb = min((int)blockIdx.x * kWN + wn, (p.N + 31) / 32 - 1);
  const int step = kWK * ksplit;
  int nb = blockIdx.y * kWK + wk;
  const uint4* wsrc = p.w + ((size_t)cb * p.NB + nb) * 128 + lane;
  const uint8_t* ssrc = p.scales + (((size_t)cb * p.NB + nb) * 16 + g) * (kPer * 4);
  const T* xsrc[kMB];
  const uint4* xp = nullptr;
  if constexpr (kPacked) {
    xp = p.xp + ((size_t)blockIdx.z * p.NB + nb) * (4 * kMB * kTerms * 32) + lane;
  } else {
#pragma unroll
    for (int j = 0; j < kMB; ++j)  // rows past the last repeat it and are not stored
      xsrc[j] = static_cast<const T*>(p.x) + (long long)min(m0 + j * 8 + g, p.M - 1) * p.xs + nb * 128 + t * 8;
  }
  struct Scales { uint32_t v[kPer]; };
  uint4 w[4];
  Scales sc[2];
  auto fetch = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(wsrc + i * 32);  // (64 rows, 16 columns): 2 x 2
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* s = ssrc + i * 8 * (kPer * 4);
      if constexpr (kPer == 1) sc[i].v[0] = __ldg(reinterpret_cast<const uint32_t*>(s));
      if constexpr (kPer == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(s));
        sc[i].v[0] = v.x; sc[i].v[1] = v.y;
      }
      if constexpr (kPer == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(s));
        sc[i].v[0] = v.x; sc[i].v[1] = v.y; sc[i].v[2] = v.z; sc[i].v[3] = v.w;
      }
    }
    wsrc += (size_t)step * 128;
    ssrc += (size_t)step * 16 * (kPer * 4);
  };
  if (nb < p.NB) fetch();
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the terms; everything before them is done
  float sum[2][kMB][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < kMB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[i][j][c] = 0.f;
  for (; nb < p.NB; nb += step) {
    uint4 cur[4];
    Scales cs[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) cur[i] = w[i];
    cs[0] = sc[0]; cs[1] = sc[1];
    if (nb + step < p.NB) fetch();
    float acc[2][kMB][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t f[kMB][kTerms][4];
      if constexpr (kPacked) {
        load_quarter<T, kTerms, kMB, true>(p, xsrc, xp + q * (kMB * kTerms * 32), 0, f);
      } else {
        const T* at[kMB];
#pragma unroll
        for (int j = 0; j < kMB; ++j) at[j] = xsrc[j] + q * 32;
        load_quarter<T, kTerms, kMB, false>(p, at, nullptr, nb * 128 + q * 32 + t * 8, f);
      }
      const bool start = q % (4 / kPer) == 0, end = (q + 1) % (4 / kPer) == 0;
      if (start) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < kMB; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = cur[(q >> 1) * 2 + i];
        uint32_t a0[4], a1[4];
        widen(q & 1 ? v.z : v.x, a0);
        widen(q & 1 ? v.w : v.y, a1);
#pragma unroll
        for (int j = 0; j < kMB; ++j)
#pragma unroll
          for (int e = kTerms - 1; e >= 0; --e) {
            mma16816(acc[i][j], a0, f[j][e][0], f[j][e][1]);
            mma16816(acc[i][j], a1, f[j][e][2], f[j][e][3]);
          }
        if (end) {
          const uint32_t u = cs[i].v[q / (4 / kPer)];
          const float s0 = __uint_as_float(u << 16), s1 = __uint_as_float(u & 0xffff0000u);
#pragma unroll
          for (int j = 0; j < kMB; ++j) {
            sum[i][j][0] = fmaf(s0, acc[i][j][0], sum[i][j][0]);
            sum[i][j][1] = fmaf(s0, acc[i][j][1], sum[i][j][1]);
            sum[i][j][2] = fmaf(s1, acc[i][j][2], sum[i][j][2]);
            sum[i][j][3] = fmaf(s1, acc[i][j][3], sum[i][j][3]);
          }
        }
      }
    }
    if constexpr (kPacked) {
      xp += (size_t)step * (4 * kMB * kTerms * 32);
    } else {
#pragma unroll
      for (int j = 0; j < kMB; ++j) xsrc[j] += step * 128;
    }
  }
  // columns of the CTA x rows, summed over its warps, then over the cluster
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < kMB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        part[(warp * 32 + i * 16 + g + (c >> 1) * 8) * kRows + j * 8 + 2 * t + (c & 1)] = sum[i][j][c];
  __syncthreads();
  auto local = [&](int n, int m) { return part + n * kRows + m; };
  if (ksplit > 1) {
    for (int e = tid; e < kCols * kMB * 8; e += kW4Warps * 32) {
      const int n = e % kCols, m = e / kCols;
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < kWK; ++i) y += *local(i * kCols + n, m);
      *local(n, m) = y;
    }
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  }
  for (int e = tid + (ksplit > 1 ? blockIdx.y * kW4Warps * 32 : 0); e < kCols * kMB * 8;
       e += kW4Warps * 32 * (ksplit > 1 ? ksplit : 1)) {
    const int n = e % kCols, m = e / kCols;
    const int col = blockIdx.x * kCols + n, row = m0 + m;
    if (col >= p.N || row >= p.M) continue;
    float y = 0.f;
    if (ksplit > 1) {
      for (int r = 0; r < ksplit; ++r) {
        uint32_t at;
        float v;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local(n, m))), "r"(r));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
        y += v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWK; ++i) y += *local(i * kCols + n, m);
    }
    if (p.bias) y += p.bias[col];
    if (p.gelu) y = gelu_tanh(y);
    if (p.res) y += ld1(static_cast<const T*>(p.res) + (long long)row * p.rs + col);
    if constexpr (sizeof(T) == 2) static_cast<__nv_bfloat16*>(p.y)[(long long)row * p.ys + col] = __float2bfloat16(y);
    else static_cast<float*>(p.y)[(long long)row * p.ys + col] = y;
  }
  if (ksplit > 1)  // the other CTAs may still read this one's sums
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

int row_blocks(int M) { return M <= 8 ? 1 : M <= 16 ? 2 : 4; }

// Whether x goes through w4_terms_kernel first.
bool use_terms(const gdn2_w4_desc* d) {
  const int el = d->dtype == GDN2_BF16 ? 2 : 4;
  if (d->K % 8 || (d->x_stride * el) % 16) return true;
  // Measured with and without: fp32 512 x 4608 3.8 / 2.5 us, 2048 x 2048 4.9 / 3.9, 4096 x 4096 7.3 / 7.7,
  // 8192 x 8192 17.4 / 24.6 (1 row) and 48 / 78 (32 rows).
  return el == 4 && (long long)d->K * d->N >= (4 << 20);
}

template <class T, int kTerms, int kMB, int kPer, bool kPacked>
cudaError_t launch_one(const W4Params& p, cudaStream_t st) {
  const int blocks = ((p.N + 31) / 32 + kMB - 1) / kMB, rows = (p.M + 8 * kMB - 1) / (8 * kMB);
  // The rows of the weight are split over a cluster while the CTAs stay within one for each SM (two for
  // 9 to 16 bf16 rows, whose CTAs fit twice) and every warp has a batch: a CTA costs about 2 us besides
  // its batches.  Measured with 1 / 2 / 8 CTAs: 16384 x 128, 4 rows 11.4 / 7.8 / 4.2 us; 8192 x 8192, 256
  // CTAs, 11.8 / 14.7 us with 1 / 2.
  const int most = kSmCount * (kTerms == 1 && kMB == 2 ? 2 : 1);
  int ks = 1;
  while (ks < 8 && blocks * rows * ks * 2 <= most && ks * (kW4Warps / kMB) < p.NB) ks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, ks, rows);
  cfg.blockDim = dim3(kW4Warps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (ks > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = 1; at[n].val.clusterDim.y = ks; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (kPacked) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, w4_kernel<T, kTerms, kMB, kPer, kPacked>, p);
}
template <class T, int kTerms, int kMB, bool kPacked>
cudaError_t launch_group(const W4Params& p, int group, cudaStream_t st) {
  if (group == 32) return launch_one<T, kTerms, kMB, 4, kPacked>(p, st);
  if (group == 64) return launch_one<T, kTerms, kMB, 2, kPacked>(p, st);
  return launch_one<T, kTerms, kMB, 1, kPacked>(p, st);
}
template <class T, int kTerms, bool kPacked>
cudaError_t launch_rows(const W4Params& p, int group, cudaStream_t st) {
  switch (row_blocks(p.M)) {
    case 1: return launch_group<T, kTerms, 1, kPacked>(p, group, st);
    case 2: return launch_group<T, kTerms, 2, kPacked>(p, group, st);
    default: return launch_group<T, kTerms, 4, kPacked>(p, group, st);
  }
}
template <class T>
cudaError_t launch(W4Params p, int group, bool terms, void* ws, cudaStream_t st) {
  constexpr int kTerms = sizeof(T) == 2 ? 1 : 3;
  if (!terms) return launch_rows<T, kTerms, false>(p, group, st);
  const int mb = row_blocks(p.M);
  const long long units = (long long)((p.M + 8 * mb - 1) / (8 * mb)) * p.NB * 4 * mb;
  w4_terms_kernel<T><<<(unsigned)((units + 7) / 8), 256, 0, st>>>(p, static_cast<uint4*>(ws), mb);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  p.xp = static_cast<const uint4*>(ws);
  return launch_rows<T, kTerms, true>(p, group, st);
}

gdn2_status check_w4(const gdn2_w4_desc* d) {
  if (!d || d->M <= 0 || d->K <= 0 || d->N <= 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->act != GDN2_ACT_NONE && d->act != GDN2_ACT_GELU_TANH) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->x_stride < 0 || d->y_stride < d->N || d->res_stride < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->group != 32 && d->group != 64 && d->group != 128) return GDN2_ERR_UNSUPPORTED;
  if (d->M > 65535 * 32 || d->K > (1 << 30) || d->N > (1 << 30)) return GDN2_ERR_UNSUPPORTED;  // rows: the grid's limit
  return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_w4_workspace_bytes(const gdn2_w4_desc* d) {
  using namespace gdn2;
  if (check_w4(d) != GDN2_OK || !use_terms(d)) return 0;
  const size_t mb = row_blocks(d->M), blocks = (d->M + 8 * mb - 1) / (8 * mb), batches = (d->K + 127) / 128;
  return blocks * batches * 4 * mb * (d->dtype == GDN2_BF16 ? 1 : 3) * 512;
}

extern "C" gdn2_status gdn2_w4_linear(const gdn2_w4_desc* d, const void* x, const void* packed, const void* scales,
                                      const float* bias, const void* residual, void* y, void* workspace,
                                      void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_w4(d);
  if (s != GDN2_OK) return s;
  const bool terms = use_terms(d);
  const void* on16[] = {x, packed, scales, terms ? workspace : x};
  for (const void* q : on16)
    if (!q || (reinterpret_cast<uintptr_t>(q) & 15u)) return GDN2_ERR_INVALID_ARGUMENT;
  if (!y) return GDN2_ERR_INVALID_ARGUMENT;
  W4Params p{};
  p.x = x;
  p.w = static_cast<const uint4*>(packed);
  p.scales = static_cast<const uint8_t*>(scales);
  p.bias = bias; p.res = residual; p.y = y;
  p.xs = d->x_stride; p.rs = d->res_stride; p.ys = d->y_stride;
  p.M = d->M; p.K = d->K; p.N = d->N;
  p.NB = (d->K + 127) / 128;
  p.gelu = d->act == GDN2_ACT_GELU_TANH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == GDN2_BF16 ? launch<__nv_bfloat16>(p, d->group, terms, workspace, st)
                                              : launch<float>(p, d->group, terms, workspace, st);
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
