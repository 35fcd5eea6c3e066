// The linear product with its epilogue, and its backward (sm_100a).
//   z = x W + b,  y = act(z) + r;    dz = dy act'(z),  db = sum over rows of dz,  dx = dz W^T,  dW = x^T dz
// x (M, K), W (K, N), y, z, r (M, N) are bf16 or fp32; sums are fp32.
//
// Small products and few rows have kernels of their own below, in plain fp32.  The others, all three of them, run on the
// 5th-generation tensor cores from bf16 operands: D (rows, cols) = A B with A and B
// read in place by tiled copies, either of them contiguous along the summed dimension or across it (W in the
// forward, x and dz for dW), so that nothing is transposed in memory.  An fp32 operand is first cut into three
// bf16 terms of 8 bits each (x = t0 + t1 + t2 to 2^-27 of x), and the six products t_i u_j with i + j <= 2 are
// summed, the small ones first: what is left out is below 2^-26 of a product.  fp32's whole range of exponents
// is kept, which two fp16 terms with a scale (half the products) would not.
// The tensor cores' additions truncate: fp32 sums leave them every 64 values of the summed dimension and go on in
// registers with rounded additions (2048 x 512 x 2048: 1e-7 of the result off; every 128 values 6e-7, 256 1.5e-6, for
// 4 to 20 % of the time; a plain fp32 product 4e-7).  bf16 sums leave them every 1024 values, so
// that what truncation takes, some 4e-6 of a sum, does not grow with its length: 2048 x K x 2048 random values are rounded to
// another bf16 value than the exact sum in 7 places of 10000 at any K (7e-5 of the result's norm); without it in 47 at K = 8192
// (2.2e-4) and in 1000 at K = 262144 (1.3e-3).  8192 x 4096 x 4096 takes 202 us for 198, with a residual 229 for 211: an
// epilogue that reads is still at work when the next turn is there to be taken out.  Every 2048 values 200 and 224 us (1e-4),
// every 4096 198 and 212 (1.5e-4 at any K above).
// An infinite or huge fp32 value makes infinities of opposite signs in its terms: a result that is NaN is summed
// again by itself from the fp32 operands, and so is what the plain sum makes of them.
//
// One CTA a SM (or a pair of CTAs on two SMs, whose tile of 256 x 256 shares the operands between them) walks
// output tiles; a warp issues the copies, one thread the products into one of two accumulators in tensor
// memory, sixteen warps empty the other one through the epilogue.  Few tiles with a long sum are split along it,
// and a second launch adds the parts in a fixed order.
//
// Measured.  bf16, 8192 x 4096 x 4096: 202 to 206 us a product, 218 with 8192 values to a sum (1.26 to 1.36 PFLOP/s; the
// products alone, without copies, 163, the copies alone 122: what is left is their overlap under the power limit).  fp32, 16384 x 512 x 2048:
// 151 to 162 us (1.3 PFLOP/s of bf16 products); the forward's epilogue writes y and z, 268 MB, and is a fifth of it:
// the warps that empty the accumulators every 64 values are the ones that write.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "gdn2_common.cuh"

namespace gdn2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kBK = 64;                 // values of the summed dimension in a stage: 128 bytes of bf16
constexpr int kEpiWarps = 16;
constexpr int kGemmThreads = 32 * (kEpiWarps + 2);
constexpr int kStageRow = 128;          // bytes

// How a result element leaves: y = act(v + bias) + residual, with v + bias kept in z.
struct Epilogue {
  void* y;
  void* z;                              // null: not kept
  const void* bias;                     // null: none
  const void* residual;                 // null: none
  long long ldr;
  long long ldy;                        // y and z
  int y_bf16, bias_bf16, act;
  float* parts;                         // not null: sums go here, (splits, rows, cols) fp32
  // the operands in fp32, for sums that are NaN; null: bf16 operands, whose sums are as they are
  const float *a, *b;
  const float *az, *bz;                 // not null: that operand is times the slope of GELU at these
  long long a_row, a_k, b_col, b_k;     // element strides
};

struct GemmParams {
  Epilogue ep;
  int rows, cols, k;
  int tiles_m, tiles_n, splits, kblocks, per_split;   // per_split: k blocks of a split
  int a_mn, b_mn;                       // contiguous across the summed dimension
  int pairs;                            // y, z and the residual may be read and written two bf16 values at a time
  uint32_t* flags;
};

// ---- activation ---------------------------------------------------------------------------------
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f;
// 0.5 z (1 + tanh u) = z / (1 + exp(-2 u)),  u = C (z + A z^3).  The approximate exponential and reciprocal leave about
// 2^-22 of the gate, and so does the rounding of the exponent above z = -1; below, it leaves 2^-20.3 at -3, 2^-18.6 at -5 and
// 2^-16.2 at -10, of gates that are 2^-10, 2^-24 and 2^-126 by then.  GELU itself is within 2^-25 and 2^-22 of its value.
__device__ __forceinline__ float gelu_gate(float z) {
  constexpr float kA = -2.f * kGeluC * 1.4426950408889634f, kB = kA * kGeluA;
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(z * fmaf(kB * z, z, kA)));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}
__device__ __forceinline__ float gelu(float z) { return z * gelu_gate(z); }
__device__ __forceinline__ float gelu_slope(float z) {
  const float s = gelu_gate(z);
  // s is 0 or 1 long before z^2 overflows, and the second term nothing
  return s + z * s * (1.f - s) * (2.f * kGeluC) * (1.f + 3.f * kGeluA * fminf(z * z, 1e38f));
}

__device__ __forceinline__ float load_f(const void* p, long long i, int bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_f(void* p, long long i, int bf16, float v) {
  if (bf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// A sum that is NaN, again from the operands themselves.
__device__ __forceinline__ float plain_sum(const Epilogue& e, long long row, long long col, int k) {
  float s = 0.f;
  for (int i = 0; i < k; ++i) {
    const long long at = row * e.a_row + i * e.a_k, bt = col * e.b_col + i * e.b_k;
    float x = e.a[at], y = e.b[bt];
    if (e.az) x *= gelu_slope(e.az[at]);
    if (e.bz) y *= gelu_slope(e.bz[bt]);
    s = fmaf(x, y, s);
    if (s != s) break;                  // and stays so
  }
  return s;
}

__device__ __forceinline__ void finish(const Epilogue& e, long long row, long long col, float v, int k, float bias) {
  if (e.a && v != v) v = plain_sum(e, row, col, k);
  v += bias;
  const long long at = row * e.ldy + col;
  if (e.z) store_f(e.z, at, e.y_bf16, v);
  if (e.act == GDN2_ACT_GELU_TANH) v = gelu(v);
  if (e.residual) v += load_f(e.residual, row * e.ldr + col, e.y_bf16);
  store_f(e.y, at, e.y_bf16, v);
}
// The rows of a column whose bit is set, `step` apart, whose sums are NaN.
__device__ __noinline__ void again(const Epilogue& e, long long row, int step, long long col, uint32_t rows, int k, float bias) {
  for (int i = 0; i < 8; ++i)
    if ((rows >> i) & 1u) finish(e, row + i * step, col, __int_as_float(0x7fc00000), k, bias);
}

// W neighbouring values (1 or 2) of T.
template <class T, int W>
struct Values {
  T x[W];
};
template <>
struct alignas(4) Values<__nv_bfloat16, 2> {
  __nv_bfloat16 x[2];
};
template <class T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
  else return v;
}
// The same for eight rows, STEP apart, of W columns; rows from `rows` on are not there (ALL: they all are).  Loads
// come first.
template <class T, int W, int STEP, bool ALL>
__device__ __forceinline__ void finish8(const Epilogue& e, float (&v)[8][W], long long row, long long col, long long rows, int k,
                                        const float (&bias)[W]) {
  using Vec = Values<T, W>;
  const int left = ALL ? 8 : (int)max(0ll, min(8ll, (rows - row + STEP - 1) / STEP));
  Vec r[8];
  if (e.residual) {
    const T* p = static_cast<const T*>(e.residual) + row * e.ldr + col;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += STEP * e.ldr)
      if (ALL || i < left) r[i] = *reinterpret_cast<const Vec*>(p);
  }
  uint32_t nan = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) nan |= (v[i][0] != v[i][0] && (ALL || i < left) ? 1u : 0u) << i;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) v[i][j] += bias[j];
  auto put = [&](void* to) {
    T* p = static_cast<T*>(to) + row * e.ldy + col;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += STEP * e.ldy) {
      Vec o;
#pragma unroll
      for (int j = 0; j < W; ++j) o.x[j] = narrow<T>(v[i][j]);
      if (ALL || i < left) *reinterpret_cast<Vec*>(p) = o;
    }
  };
  if (e.z) put(e.z);
  if (e.act == GDN2_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) v[i][j] = gelu(v[i][j]);
  }
  if (e.residual) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) v[i][j] += to_f<T>(r[i].x[j]);
  }
  put(e.y);
  if (nan && e.a) again(e, row, STEP, col, nan, k, bias[0]);
}

// ---- the product --------------------------------------------------------------------------------
template <int CG, int P>
struct Gemm {
  static constexpr int kTileM = 128 * CG, kTileN = 128 * CG;        // of the CTA or the pair
  static constexpr int kOperand = 128 * kStageRow;                  // a CTA's part of one term of A or of B
  static constexpr int kStage = 2 * P * kOperand;
  static constexpr int kStages = P == 1 ? 5 : 2;
  static constexpr int kTmem = 2 * kTileN;                          // two accumulators' columns
  static constexpr int kCols = P == 1 ? 32 : 16;                    // columns that a warp turns around at a time
  static constexpr int kTurn = P == 1 ? 16 : 1;                     // blocks of the sum in an accumulator's turn
  static constexpr size_t kStaging = kEpiWarps * 32 * kCols * sizeof(float);
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kStaging + 256;
};

// A wait that ends: after kWaitCycles, or once another of this CTA's waits has run out.
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, volatile int* dead, uint32_t* flags) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*dead) return false;
    if ((it & 255u) == 255u && clock64() - t0 > kWaitCycles) {
      *dead = 1;
      if (flags) flags[2] = 1;
      return false;
    }
  }
}

__device__ __forceinline__ uint32_t leader_addr(const void* p) {    // the same place in the cluster's CTA 0
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
template <int CG>
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
  else
    mma_t<kBF16>(d, a, b, id, accumulate);
}
// Arrives at the barrier of every CTA of the pair once the products issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    mma_commit(bar);
}
// Operand descriptors, 128-byte swizzle.  Contiguous along the sum: rows of 128 bytes, eight rows (1024 bytes) an
// atom, 16 values further 32 bytes on.  Contiguous across it: blocks of 64 across x 64 along, `group` bytes apart;
// eight values along the sum are 1024 bytes, 16 are 2048.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn, uint32_t group) {
  return sdesc(addr, mn ? group : 16u, 1024u) | ((uint64_t)2u << 61);
}

struct Work {
  int tm, tn, kb0, kb1, split;
};
__device__ __forceinline__ Work work_of(const GemmParams& p, int i) {
  Work w;
  const int tiles = p.tiles_m * p.tiles_n;
  w.split = i / tiles;
  const int t = i - w.split * tiles;
  // bands of 16 tiles down the rows: the CTAs at work at a time share both operands in L2
  const int band = t / (16 * p.tiles_n), first = band * 16, high = min(16, p.tiles_m - first);
  const int in = t - band * 16 * p.tiles_n;
  w.tm = first + in % high;
  w.tn = in / high;
  w.kb0 = w.split * p.per_split;
  w.kb1 = min(p.kblocks, w.kb0 + p.per_split);
  return w;
}

// What an epilogue warp does with the accumulators' turns: `acc` is the one whose turn it is, `phase` the turn's parity.
struct Turns {
  uint64_t *full, *empty;
  volatile int* dead;
  uint32_t* flags;
  uint32_t tmem, col0;                  // the warp's first column
  __device__ __forceinline__ void wait(uint32_t acc, uint32_t phase) const {
    bounded_wait(&full[acc], phase, dead, flags);
    __syncwarp();
    tc_fence_after();
  }
  template <int CG>
  __device__ __forceinline__ void release(uint32_t& acc, uint32_t& phase) const {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      if constexpr (CG == 2)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(&empty[acc])) : "memory");
      else
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[acc])) : "memory");
    }
    acc ^= 1u;
    if (!acc) phase ^= 1u;
  }
  // A sum's turns added up, in the last one's accumulator: the epilogue needs the registers.
  template <int CG, int P>
  __device__ __forceinline__ void add(int blocks, uint32_t& acc, uint32_t& phase) const {
    using G = Gemm<CG, P>;
    constexpr int kQuarter = G::kTileN / 4;
    float sum[kQuarter];
#pragma unroll
    for (int j = 0; j < kQuarter; ++j) sum[j] = 0.f;
    for (int k = G::kTurn;; k += G::kTurn) {
      wait(acc, phase);
#pragma unroll
      for (int c = 0; c < kQuarter; c += 16) {
        float v[16];
        tmem_ld16(tmem + acc * G::kTileN, col0 + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[c + j] += v[j];
      }
      if (k >= blocks) break;
      release<CG>(acc, phase);
    }
#pragma unroll
    for (int c = 0; c < kQuarter; c += 16) tmem_st16(tmem + acc * G::kTileN, col0 + c, sum + c);
  }
};

// LONG: sums of several turns.  A kernel of its own, so that sums of one turn keep their registers: 8192 x 4096 x 4096 in one
// turn 193 us, 195.5 where the code for several stood beside it.  (One CTA a SM: for two the compiler leaves it 56 registers.)
template <int CG, int P, bool LONG>
__global__ void __launch_bounds__(kGemmThreads, LONG && P == 1 ? 1 : 0)
    linear_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ GemmParams p) {
  using G = Gemm<CG, P>;
  extern __shared__ uint8_t raw[];
  uint8_t* stages = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  float* staging = reinterpret_cast<float*>(stages + (size_t)G::kStages * G::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(staging) + G::kStaging);
  uint64_t* empty = full + G::kStages;
  uint64_t* acc_full = empty + G::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_at + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? blockIdx.x & 1 : 0;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    for (int i = 0; i < G::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps * CG);
    }
    *dead = 0;
    fence_mbar_init();
  }
  if (warp == kEpiWarps + 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)),
                   "r"(G::kTmem) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_at, G::kTmem);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cg::this_cluster().sync();
  tc_fence_after();
  pdl_enter();                          // from here on what the kernel before wrote is read
  const uint32_t tmem = *tmem_at;
  const int items = p.tiles_m * p.tiles_n * p.splits, stride = gridDim.x / CG;
  const uint32_t group = P * 8192;      // 64 values across the sum of all terms, contiguous across

  if (warp == kEpiWarps) {
    if (lane == 0) {  // copies
      uint32_t stage = 0, phase = 0;
      bool fine = true;
      for (int it = blockIdx.x / CG; it < items && fine; it += stride) {
        const Work w = work_of(p, it);
        const int m0 = w.tm * G::kTileM + rank * 128, n0 = w.tn * G::kTileN + rank * 128;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!(fine = bounded_wait(&empty[stage], phase ^ 1u, dead, p.flags))) break;
          const uint32_t bar = CG == 2 ? leader_addr(&full[stage]) : smem_u32(&full[stage]);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], G::kStage * CG);
          const uint32_t a = smem_u32(stages + (size_t)stage * G::kStage), b = a + P * G::kOperand;
          const int k0 = kb * kBK;
          if (p.a_mn) {
            tile_load<CG>(a, &map_a, m0, k0, bar);
            tile_load<CG>(a + group, &map_a, m0 + 64, k0, bar);
          } else {
            tile_load<CG>(a, &map_a, k0, m0, bar);
          }
          if (p.b_mn) {
            tile_load<CG>(b, &map_b, n0, k0, bar);
            tile_load<CG>(b + group, &map_b, n0 + 64, k0, bar);
          } else {
            tile_load<CG>(b, &map_b, k0, n0, bar);
          }
          if (++stage == G::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // No copy is in flight when the CTA ends: every stage was consumed, or a wait ran out, and then what was
      // issued is given its time.
      for (int i = 0; i < G::kStages && fine; ++i) {
        fine = bounded_wait(&empty[stage], phase ^ 1u, dead, p.flags);
        if (++stage == G::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!fine) {
        const long long t0 = clock64();
        while (clock64() - t0 < 20 * 1000 * 1000) __nanosleep(1000);
      }
    }
  } else if (warp == kEpiWarps + 1) {
    if (lane == 0 && rank == 0) {  // products
      const uint32_t id = (idesc(kBF16, G::kTileN, p.a_mn, p.b_mn, false) & ~(31u << 24)) | (uint32_t)(G::kTileM >> 4) << 24;
      const uint32_t step_a = (p.a_mn ? 2048u : 32u) >> 4, step_b = (p.b_mn ? 2048u : 32u) >> 4;
      const uint32_t term_a = (p.a_mn ? 8192u : (uint32_t)G::kOperand) >> 4, term_b = (p.b_mn ? 8192u : (uint32_t)G::kOperand) >> 4;
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool fine = true;
      for (int it = blockIdx.x / CG; it < items && fine; it += stride) {
        const Work w = work_of(p, it);
        for (int kb = w.kb0; kb < w.kb1 && fine; ++kb) {
          const int turn = (kb - w.kb0) % G::kTurn;
          const bool first = turn == 0;                  // of an accumulator's turn
          if (first && !(fine = bounded_wait(&acc_empty[acc], acc_phase ^ 1u, dead, p.flags))) break;
          if (!(fine = bounded_wait(&full[stage], phase, dead, p.flags))) break;
          tc_fence_after();
          const uint32_t d = tmem + acc * G::kTileN;
          const uint32_t sa = smem_u32(stages + (size_t)stage * G::kStage);
          const uint64_t a = operand_desc(sa, p.a_mn, group), b = operand_desc(sa + P * G::kOperand, p.b_mn, group);
          uint32_t add = first ? 0u : 1u;
          if constexpr (P == 3) {
            constexpr int kA[6] = {2, 1, 0, 1, 0, 0}, kB[6] = {0, 1, 2, 0, 1, 0};  // terms, small products first
#pragma unroll
            for (int c = 0; c < 6; ++c)
#pragma unroll
              for (int s = 0; s < kBK / 16; ++s) {
                mma_bf16<CG>(d, a + kA[c] * term_a + s * step_a, b + kB[c] * term_b + s * step_b, id, add);
                add = 1u;
              }
          } else {
#pragma unroll
            for (int s = 0; s < kBK / 16; ++s) {
              mma_bf16<CG>(d, a + s * step_a, b + s * step_b, id, add);
              add = 1u;
            }
          }
          commit<CG>(&empty[stage]);
          if (++stage == G::kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (turn == G::kTurn - 1 || kb == w.kb1 - 1) {
            commit<CG>(&acc_full[acc]);
            acc ^= 1u;
            if (!acc) acc_phase ^= 1u;
          }
        }
      }
    }
  } else {  // epilogue: warp w has rows 32 (w % 4).. and quarter w / 4 of the columns
    constexpr int kQuarter = G::kTileN / 4;
    float* mine = staging + warp * 32 * G::kCols;
    const uint32_t col0 = (warp >> 2) * kQuarter;
    const int half = lane >> 4, in = lane & 15;
    uint32_t acc = 0, acc_phase = 0;
    for (int it = blockIdx.x / CG; it < items; it += stride) {
      const Work w = work_of(p, it);
      const long long row0 = (long long)w.tm * G::kTileM + rank * 128 + (warp & 3) * 32;
      const long long out0 = (long long)w.tn * G::kTileN + col0;
      if (p.ep.residual && row0 + lane < p.rows && out0 < p.cols) {  // on its way to L2 while the products run
        const size_t el = P == 1 ? 2 : 4;
        const char* r = static_cast<const char*>(p.ep.residual) + ((row0 + lane) * p.ep.ldr + out0) * el;
        const int bytes = (int)(min((long long)kQuarter, p.cols - out0) * el);
        for (int i = 0; i < bytes; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(r + i));
      }
      // 32 rows x 16 or 32 columns at a time: from rows to lanes through shared memory, so that half a warp reads and
      // writes 16 neighbouring columns (bf16: 16 pairs) of a row; permuted there by the row, so that no two lanes
      // meet in a bank
      const bool all_rows = row0 + 32 <= p.rows;
      auto put = [&](const float* v, int c) __attribute__((always_inline)) {
        using T = std::conditional_t<P == 1, __nv_bfloat16, float>;
        constexpr int W = P == 1 ? 2 : 1, kRow = 16 * W;
        using Pair = Values<float, W>;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          Pair q;
#pragma unroll
          for (int u = 0; u < W; ++u) q.x[u] = v[W * j + u];
          *reinterpret_cast<Pair*>(mine + lane * kRow + W * (j ^ (P == 1 ? lane & 15 : lane >> 1))) = q;
        }
        __syncwarp();
        const long long col = out0 + c + W * in;
        if (col < p.cols) {
          float bias[W];
#pragma unroll
          for (int u = 0; u < W; ++u)
            bias[u] = p.ep.bias && !p.ep.parts && col + u < p.cols ? load_f(p.ep.bias, col + u, p.ep.bias_bf16) : 0.f;
#pragma unroll
          for (int i0 = half; i0 < 32; i0 += 16) {
            float u[8][W];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i0 + 2 * i;
              const Pair q = *reinterpret_cast<const Pair*>(mine + r * kRow + W * (in ^ (P == 1 ? r & 15 : r >> 1)));
#pragma unroll
              for (int x = 0; x < W; ++x) u[i][x] = q.x[x];
            }
            if (p.ep.parts) {
              float* q = p.ep.parts + ((long long)w.split * p.rows + row0 + i0) * p.cols + col;
#pragma unroll
              for (int i = 0; i < 8; ++i, q += 2 * (long long)p.cols)
                if (row0 + i0 + 2 * i < p.rows) {
#pragma unroll
                  for (int x = 0; x < W; ++x)
                    if (col + x < p.cols) q[x] = u[i][x];
                }
            } else if (W == 1 || p.pairs) {
              if (all_rows) finish8<T, W, 2, true>(p.ep, u, row0 + i0, col, p.rows, p.k, bias);
              else finish8<T, W, 2, false>(p.ep, u, row0 + i0, col, p.rows, p.k, bias);
            } else {  // rows that start on odd places: one column after the other
#pragma unroll
              for (int x = 0; x < W; ++x) {
                float one[8][1];
                const float b1[1] = {bias[x]};
#pragma unroll
                for (int i = 0; i < 8; ++i) one[i][0] = u[i][x];
                if (col + x < p.cols) finish8<T, 1, 2, false>(p.ep, one, row0 + i0, col + x, p.rows, p.k, b1);
              }
            }
          }
        }
        __syncwarp();
      };
      const Turns turns{acc_full, acc_empty, dead, p.flags, tmem, col0};
      if constexpr (LONG) turns.template add<CG, P>(w.kb1 - w.kb0, acc, acc_phase);
      else turns.wait(acc, acc_phase);
      if constexpr (P == 3) {
#pragma unroll 1
        for (int c = 0; c < kQuarter; c += 16) {
          float v[16];
          tmem_ld16(tmem + acc * G::kTileN, col0 + c, v);
          if (c + 16 == kQuarter) turns.template release<CG>(acc, acc_phase);
          put(v, c);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kQuarter; c += 32) {
          float v[32];
          tmem_ld32(tmem + acc * G::kTileN, col0 + c, v);
          if (c + 32 == kQuarter) turns.template release<CG>(acc, acc_phase);
          put(v, c);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cg::this_cluster().sync();  // the pair's products and arrivals are over
  tc_fence_after();
  if (warp == kEpiWarps + 1) {
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::kTmem) : "memory");
    else
      tmem_dealloc(tmem, G::kTmem);
  }
}

// Adds the parts of a split sum in their order and finishes: 32 neighbouring columns to a warp, four rows to a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) linear_join_kernel(const float* parts, int splits, int rows, int cols, int k,
                                                          int col_blocks, const __grid_constant__ Epilogue e) {
  pdl_enter();
  const long long n = (long long)rows * cols;
  const int block = blockIdx.x / col_blocks;
  const long long row = block * 64ll + (threadIdx.x >> 5), col = (blockIdx.x - block * col_blocks) * 32ll + (threadIdx.x & 31);
  if (col >= cols) return;
  const float* q = parts + row * cols + col;
  float v[8][1];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i][0] = row + 8 * i < rows ? q[8ll * i * cols] : 0.f;
  for (int s = 1; s < splits; ++s) {
    q += n;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i][0] += row + 8 * i < rows ? q[8ll * i * cols] : 0.f;
  }
  const float bias[1] = {e.bias ? load_f(e.bias, col, e.bias_bf16) : 0.f};
  finish8<std::conditional_t<BF16, __nv_bfloat16, float>, 1, 8, false>(e, v, row, col, rows, k, bias);
}

// ---- operands in the form that the copies need --------------------------------------------------
// Eight neighbouring values of a row, zeros past its end; `whole`: eight that may be read 16 bytes at a time.  bf16 rows
// that start anywhere are read 4 bytes at a time all the same, and shifted where they start between two words.
template <class T>
__device__ __forceinline__ void load8(const T* p, float v[8], bool whole, int left) {
  if (sizeof(T) == 2 && !whole && left > 8) {
    const bool off = reinterpret_cast<uintptr_t>(p) & 2u;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) - (off ? 2 : 0));
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(q + i);
    w[4] = off ? __ldg(q + 4) : 0u;     // up to the ninth value
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = off ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
      v[2 * i] = __uint_as_float(u << 16);
      v[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
    }
  } else if (whole) {
    if constexpr (sizeof(T) == 4) {
      ld4(p, v);
      ld4(p + 4, v + 4);
    } else {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? ld1(p + i) : 0.f;
  }
}
// Their terms: three of an fp32 value, `term` elements apart, or the bf16 value itself.
template <class T>
__device__ __forceinline__ void store_terms(__nv_bfloat16* o, long long term, float v[8]) {
#pragma unroll
  for (int t = 0; t < (sizeof(T) == 2 ? 1 : 3); ++t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      v[2 * i] -= __uint_as_float(w[i] << 16);
      v[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
    }
    *reinterpret_cast<uint4*>(o + t * term) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <class T>
__device__ __forceinline__ bool by16(const T* p, long long ld) {
  return ld % (16 / (int)sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

// (16384 x 512 fp32: 14 us for 84 MB of operands and terms; they are written to L2 and read from there.)
// rows x cols of T with rows `ld` apart -> terms of bf16, rows `ldt` apart, terms rows * ldt apart: an fp32 matrix
// in three terms, or a bf16 matrix whose rows are not on 16 bytes as it is.  Two matrices a launch.
struct TermsJob {
  const void* x;
  __nv_bfloat16* out;
  long long ld, ldt, items;             // items: groups of eight columns of all rows
  int rows, cols;
};
template <class T>
__global__ void __launch_bounds__(256) linear_terms_kernel(const __grid_constant__ TermsJob j0,
                                                           const __grid_constant__ TermsJob j1) {
  const long long all = j0.items + j1.items;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const bool second = i >= j0.items;
    const TermsJob& j = second ? j1 : j0;
    const long long at = second ? i - j0.items : i, per = j.ldt / 8, r = at / per;
    const int c = (int)(at - r * per) * 8;
    const T* x = static_cast<const T*>(j.x) + r * j.ld + c;
    float v[8];
    load8<T>(x, v, c + 8 <= j.cols && by16(static_cast<const T*>(j.x), j.ld), j.cols - c);
    store_terms<T>(j.out + r * j.ldt + c, (long long)j.rows * j.ldt, v);
  }
}

// dz = dy act'(z) (or dy) in the same form, and db's parts: a CTA takes 64 columns of `band` rows, 8 threads beside
// one another a row's.  HBM bounds it (16384 x 2048 fp32 with GELU: 78 us for 470 MB; bf16 sums alone, 8192 x 4096: 23 us
// for 67 MB).
template <class T, bool ACT>
__global__ void __launch_bounds__(256) linear_dz_kernel(const T* dy, const T* z, int rows, int cols, int band, int col_blocks,
                                                        __nv_bfloat16* out, long long ldt, float* parts) {
  __shared__ float sums[32][64 + 4];
  const int in_band = blockIdx.x / col_blocks, c0 = (blockIdx.x - in_band * col_blocks) * 64;
  const int tc = (threadIdx.x & 7) * 8, tr = threadIdx.x >> 3, c = c0 + tc;
  const long long r0 = (long long)in_band * band, r1 = min((long long)rows, r0 + band), term = rows * ldt;
  const bool whole = c + 8 <= cols && by16(dy, cols) && (!ACT || by16(z, cols));
  float s[8] = {};
#pragma unroll(ACT ? 2 : 4)
  for (long long r = r0 + tr; r < r1; r += 32) {
    float v[8], u[8];
    load8<T>(dy + r * cols + c, v, whole, cols - c);
    if constexpr (ACT) {
      load8<T>(z + r * cols + c, u, whole, cols - c);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= gelu_slope(u[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += v[i];
    if (out && c < ldt) store_terms<T>(out + r * ldt + c, term, v);
  }
  if (!parts) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[tr][tc + i] = s[i];
  __syncthreads();
  if (threadIdx.x < 64 && c0 + (int)threadIdx.x < cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sums[i][threadIdx.x];
    parts[(long long)in_band * cols + c0 + threadIdx.x] = t;
  }
}
// The bands' sums of a column: 32 columns to a CTA, eight threads to a column.
__global__ void __launch_bounds__(256) linear_db_kernel(const float* parts, int bands, int cols, void* db, int bf16) {
  __shared__ float sums[8][32];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int i = warp; i < bands; i += 8) s += parts[(long long)i * cols + c];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sums[i][lane];
  store_f(db, c, bf16, s);
}

// ---- few rows -----------------------------------------------------------------------------------
// Up to 8 rows of x a launch: W is read once, straight into fp32 products.  A CTA takes 32 V columns and a stretch of
// the sum, its eight warps and the CTAs of a cluster shares of it; their parts meet in shared memory.  The loads of W
// bound it (1 x 4096 x 4096 fp32: 10.9 us, 6.2 TB/s; 1 x 512 x 4608: 5.0 us, launch and two cluster barriers): four rows of it (bf16:
// eight) are on their way while as many are multiplied, and the first ones before x is looked at.
constexpr int kFewStretch = 256;
template <class T>
constexpr int kFewBatch = 16 / (int)sizeof(T);

struct FewParams {
  Epilogue ep;
  const void *x, *w;
  long long ldx, ldw;
  int rows, cols, k, clusters;
};
// V values of a row of W as they are in memory: 4 of bf16 in two registers.
template <class T, int V>
struct Raw {
  float x[V];
  __device__ __forceinline__ void load(const T* p, bool whole, int left) {
    if (whole) {
      if constexpr (V == 4) ld4(p, x);
      else x[0] = ld1(p);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = j < left ? ld1(p + j) : 0.f;
    }
  }
  __device__ __forceinline__ void get(float v[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = x[j];
  }
};
template <>
struct Raw<__nv_bfloat16, 4> {
  uint2 x;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool whole, int left) {
    if (whole) {
      x = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = j < left ? __ldg(reinterpret_cast<const unsigned short*>(p) + j) : 0u;
      x = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
  }
  __device__ __forceinline__ void get(float v[4]) const {
    v[0] = __uint_as_float(x.x << 16);
    v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16);
    v[3] = __uint_as_float(x.y & 0xffff0000u);
  }
};
template <class T, int V, int R>
__global__ void __launch_bounds__(256) linear_few_kernel(const __grid_constant__ FewParams p) {
  __shared__ __align__(16) float xs[kFewStretch][R];
  __shared__ __align__(16) float part[8][R][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % p.clusters, c = (blockIdx.x / p.clusters * 32 + lane) * V;
  const int share = (p.k + p.clusters - 1) / p.clusters, k0 = rank * share, k1 = min(p.k, k0 + share);
  const T* w = static_cast<const T*>(p.w) + c;
  const T* x = static_cast<const T*>(p.x);
  const int left = p.cols - c;
  const bool whole = left >= V && (V == 1 || (p.ldw % V == 0 && (reinterpret_cast<uintptr_t>(p.w) % (V * sizeof(T))) == 0));
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[r][i] = 0.f;
  for (int s = k0; s < k1; s += kFewStretch) {
    const int n = min(kFewStretch, k1 - s);
    constexpr int U = kFewBatch<T>;
    Raw<T, V> now[U], next[U];
    auto load = [&](int j0, Raw<T, V>* v) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j0 + 8 * u < n && left > 0) v[u].load(w + (long long)(s + j0 + 8 * u) * p.ldw, whole, left);
    };
    load(warp, now);
    __syncthreads();                    // xs was read
    for (int i = threadIdx.x; i < R * n; i += 256) {
      const int r = i / n, j = i - r * n;
      xs[j][r] = r < p.rows ? to_f<T>(x[r * p.ldx + s + j]) : 0.f;
    }
    __syncthreads();
    for (int j0 = warp; j0 < n; j0 += 8 * U) {
      load(j0 + 8 * U, next);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + 8 * u;
        if (j < n && left > 0) {
          float xr[R], v[V];
          now[u].get(v);
          if constexpr (R % 4 == 0) {
#pragma unroll
            for (int r = 0; r < R; r += 4) *reinterpret_cast<float4*>(xr + r) = *reinterpret_cast<const float4*>(&xs[j][r]);
          } else {
#pragma unroll
            for (int r = 0; r < R; ++r) xr[r] = xs[j][r];
          }
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[r][i] = fmaf(xr[r], v[i], acc[r][i]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(&part[warp][r][lane * 4]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    else part[warp][r][lane] = acc[r][0];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * 32 * V; i += 256) {
    const int r = i / (32 * V), j = i % (32 * V);
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += part[u][r][j];
    part[0][r][j] = s;
  }
  if (p.clusters > 1) cg::this_cluster().sync();
  else __syncthreads();
  for (int i = threadIdx.x + rank * 256; i < p.rows * 32 * V; i += 256 * p.clusters) {
    const int r = i / (32 * V), j = i % (32 * V), col = blockIdx.x / p.clusters * 32 * V + j;
    if (col >= p.cols) continue;
    float s = part[0][r][j];
    if (p.clusters > 1) {
      float q[8];                       // all on their way at once
#pragma unroll
      for (int u = 0; u < 8; ++u) q[u] = u < p.clusters ? cg::this_cluster().map_shared_rank(&part[0][r][j], u)[0] : 0.f;
      s = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += q[u];
    }
    finish(p.ep, r, col, s, p.k, p.ep.bias ? load_f(p.ep.bias, col, p.ep.bias_bf16) : 0.f);
  }
  if (p.clusters > 1) cg::this_cluster().sync();  // a CTA's parts are read until here
}

// ---- small products -----------------------------------------------------------------------------
// Where launches cost more than the products: one launch for a forward, one for dx, dW and db together, fp32 products
// of 32 x 32 tiles from shared memory, dz made as it is read (which sizes, and what both ways take: small_within).
// Eight groups of 64 threads share a tile's sum, 4 x 4 of its elements a thread, and join at the end in their order.  A
// step of 64 along the sum takes 1.0 us: the loads' and shared memory's latency, with a tile's 16 warps alone on their SM
// and half of its issue slots empty (four groups, 8 warps: 1.05 us, in bf16 1.3).
constexpr int kSmallTile = 32, kSmallK = 64, kSmallRow = kSmallTile + 4, kSmallThreads = 512,
              kSmallGroups = kSmallThreads / 64, kSmallLoads = kSmallTile * kSmallK / kSmallThreads;
static_assert(kSmallTile == 32 && kSmallThreads == 512 && kSmallLoads == 4, "SmallOperand");
struct Product {
  const void *a, *b;                    // rows x k and k x cols
  const void* z;                        // not null: a (b where z_of_b) is times the slope of GELU at these
  long long a_row, a_k, b_k, b_col;     // element strides: of each pair one is 1
  int rows, cols, k, z_of_b;
  Epilogue ep;
  void* sums;                           // sums over k of b's columns, or null
  int sums_bf16;
};
struct Products {
  Product p[2];
  int tiles0;                           // of p[0]; the other tiles are p[1]'s
};
// One operand's elements of a k-tile: element j of a thread is at i = i0 + di (j % 2), k = kb + dk (j % 2) + 32 (j / 2),
// so that a warp reads along the stride of one.  In shared memory element (k, i) stands at k rows and i ^ (k / 8 % 4):
// without bank conflicts along either, and four elements of 16 bytes stay together.
struct SmallOperand {
  long long at, step, pitch, pitch2;
  int kb, dk, left, di, slot;
  bool along;
  __device__ __forceinline__ SmallOperand(long long s_i, long long s_k, int i0, int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    along = s_k == 1;                   // lanes along k
    const int i = along ? warp : lane;
    kb = along ? lane : warp;
    at = (i0 + i) * s_i + kb * s_k;
    step = kSmallK * s_k;
    pitch = 16 * (along ? s_i : s_k);
    pitch2 = 32 * s_k;
    dk = along ? 0 : 16;
    di = along ? 16 : 0;
    left = n - i0 - i;
    slot = along ? lane * kSmallRow + (warp ^ (lane >> 3)) : warp * kSmallRow + (lane ^ (warp >> 3));
  }
  template <class T>
  __device__ __forceinline__ void load(T (&v)[kSmallLoads], const void* p, int k) const {
#pragma unroll
    for (int j = 0; j < kSmallLoads; ++j)
      v[j] = left > di * (j & 1) && kb + dk * (j & 1) + 32 * (j >> 1) < k
                 ? static_cast<const T*>(p)[at + (j & 1) * pitch + (j >> 1) * pitch2] : T(0.f);
  }
  __device__ __forceinline__ void keep(const float (&v)[kSmallLoads], float* s) const {
#pragma unroll
    for (int j = 0; j < kSmallLoads; ++j)
      s[(along ? slot + 16 * (j & 1) : (slot ^ 2 * (j & 1)) + 16 * (j & 1) * kSmallRow) + 32 * (j >> 1) * kSmallRow] = v[j];
  }
};
template <class T>
__global__ void __launch_bounds__(kSmallThreads) linear_small_kernel(const __grid_constant__ Products both) {
  __shared__ __align__(16) float tiles[2][2][kSmallK * kSmallRow];
  const bool second = (int)blockIdx.x >= both.tiles0;
  const Product& p = both.p[second];
  const int tile = second ? blockIdx.x - both.tiles0 : blockIdx.x, tiles_n = (p.cols + kSmallTile - 1) / kSmallTile;
  const int row0 = tile / tiles_n * kSmallTile, col0 = tile % tiles_n * kSmallTile;
  const int group = threadIdx.x >> 6, ty = (threadIdx.x >> 3) & 7, tx = threadIdx.x & 7;
  SmallOperand oa(p.a_row, p.a_k, row0, p.rows), ob(p.b_col, p.b_k, col0, p.cols);
  const void *pa = p.a, *pb = p.b, *pz = p.z;
  const bool z_of_b = p.z_of_b, sums = p.sums && row0 == 0;
  T ra[kSmallLoads], rb[kSmallLoads], rz[kSmallLoads];
  auto load = [&](int k) {
    oa.load(ra, pa, k);
    ob.load(rb, pb, k);
    if (pz) {
      if (z_of_b) ob.load(rz, pz, k);
      else oa.load(rz, pz, k);
    }
    oa.at += oa.step;
    ob.at += ob.step;
  };
  float acc[4][4] = {}, sum[4] = {};
  load(p.k);
  int s = 0;
  for (int k = p.k; k > 0; k -= kSmallK, s ^= 1) {
    float va[kSmallLoads], vb[kSmallLoads];
#pragma unroll
    for (int j = 0; j < kSmallLoads; ++j) {
      va[j] = to_f<T>(ra[j]);
      vb[j] = to_f<T>(rb[j]);
    }
    if (pz) {
#pragma unroll
      for (int j = 0; j < kSmallLoads; ++j) {
        const float slope = gelu_slope(to_f<T>(rz[j]));
        if (z_of_b) vb[j] *= slope;
        else va[j] *= slope;
      }
    }
    oa.keep(va, tiles[s][0]);
    ob.keep(vb, tiles[s][1]);
    __syncthreads();                    // the other stage was read before the last one of these
    if (k > kSmallK) load(k - kSmallK);
    const float *as = tiles[s][0] + group * kSmallRow + 4 * ty, *bs = tiles[s][1] + group * kSmallRow + 4 * tx;
#pragma unroll
    for (int q = 0; q < kSmallK / kSmallGroups; ++q) {      // k = 8 q + group
      const float4 x4 = *reinterpret_cast<const float4*>(as + kSmallGroups * q * kSmallRow), y4 = *reinterpret_cast<const float4*>(bs + kSmallGroups * q * kSmallRow);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i ^ (q & 3)], y[j ^ (q & 3)], acc[i][j]);
      if (sums)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += y[j ^ (q & 3)];
    }
  }
  __syncthreads();
  float* join = tiles[0][0];            // 8 groups of 32 x 32 sums, then 8 of 32
  constexpr int kAll = kSmallTile * kSmallTile;
  static_assert(sizeof(tiles) >= 4 * kSmallGroups * (kAll + kSmallTile), "join");
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4*>(join + group * kAll + (4 * ty + i) * kSmallTile + 4 * tx) =
        make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  if (sums && ty == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j) join[kSmallGroups * kAll + group * kSmallTile + 4 * tx + j] = sum[j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAll / kSmallThreads; ++i) {
    const int e = threadIdx.x + kSmallThreads * i, row = row0 + e / kSmallTile, col = col0 + e % kSmallTile;
    if (row < p.rows && col < p.cols) {
      float v = 0.f;
#pragma unroll
      for (int g = 0; g < kSmallGroups; ++g) v += join[g * kAll + e];
      finish(p.ep, row, col, v, p.k, p.ep.bias ? load_f(p.ep.bias, col, p.ep.bias_bf16) : 0.f);
    }
  }
  if (sums && threadIdx.x < kSmallTile && col0 + (int)threadIdx.x < p.cols) {
    float v = 0.f;
#pragma unroll
    for (int g = 0; g < kSmallGroups; ++g) v += join[kSmallGroups * kAll + g * kSmallTile + threadIdx.x];
    store_f(p.sums, col0 + threadIdx.x, p.sums_bf16, v);
  }
}

// ---- host ---------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// A bf16 matrix (terms of it `term` elements apart), outer x inner, rows `ld` elements apart.
struct Operand {
  const void* p;
  long long outer, inner, ld, term;
  bool mn;                              // the summed dimension is the outer one
};
bool make_map(CUtensorMap* m, const Operand& o, int terms) {
  const EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer, (cuuint64_t)terms};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(terms > 1 ? o.term : o.ld * o.outer) * 2};
  const cuuint32_t box[3] = {64, o.mn ? 64u : 128u, (cuuint32_t)terms}, unit[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box, unit,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  return encode() || (bind_context(), encode());
}

constexpr int kSMs = 148;
struct GemmPlan {
  int cg, tiles_m, tiles_n, kblocks, splits, per_split;
};
GemmPlan plan_gemm(long long rows, long long cols, long long k, int terms) {
  const int terms_cost = terms == 3 ? 6 : 1;
  GemmPlan g{};
  g.kblocks = (int)((k + kBK - 1) / kBK);
  // Single CTAs or pairs, by what the busiest SM has to do: a block of the sum takes a pair 512 cycles and a
  // single CTA, whose operands come from L2 and shared memory twice as often, about 320 (measured 500 to 700); an
  // epilogue of 128 columns about 3000.  (bf16, 777 x 1001 x 2503: 22.5 us as 40 pairs, 15.6 as 140 CTAs.)
  long long best = 0;
  for (int cg = 1; cg <= 2; ++cg) {
    const int t = 128 * cg, workers = kSMs / cg;
    const long long tm = (rows + t - 1) / t, tn = (cols + t - 1) / t, n = tm * tn;
    long long s = 1;
    if (2 * n <= workers) {
      s = workers / n;
      if (s > g.kblocks / 4) s = g.kblocks / 4;
      if (s > 16) s = 16;
      if (s < 1) s = 1;
    }
    const long long waves = (n * s + workers - 1) / workers, blocks = (g.kblocks + s - 1) / s;
    const long long cost = waves * (blocks * (cg == 2 ? 512 : 320) * terms_cost + 3000 * cg);
    if (cg == 1 || cost < best) {
      best = cost;
      g.cg = cg;
      g.tiles_m = (int)tm;
      g.tiles_n = (int)tn;
      g.splits = (int)s;
    }
  }
  g.per_split = (g.kblocks + g.splits - 1) / g.splits;
  g.splits = (g.kblocks + g.per_split - 1) / g.per_split;
  return g;
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t parts_of(const GemmPlan& g, long long rows, long long cols) {
  return g.splits > 1 ? round256((size_t)g.splits * rows * cols * sizeof(float)) : 0;
}

template <int CG, int P, bool LONG>
cudaError_t launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, cudaStream_t st) {
  using G = Gemm<CG, P>;
  static unsigned long long done = 0;
  cudaError_t e = smem_attr_once(linear_gemm_kernel<CG, P, LONG>, (int)G::kSmem, done);
  if (e != cudaSuccess) return e;
  const int items = p.tiles_m * p.tiles_n * p.splits, workers = kSMs / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((items < workers ? items : workers) * CG));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, linear_gemm_kernel<CG, P, LONG>, a, b, p);
}

// One product; `parts` has parts_of() bytes.
cudaError_t gemm(const Operand& a, const Operand& b, int terms, Epilogue ep, long long rows, long long cols, long long k,
                 float* parts, uint32_t* flags, cudaStream_t st) {
  const GemmPlan g = plan_gemm(rows, cols, k, terms);
  CUtensorMap ma, mb;
  if (!make_map(&ma, a, terms) || !make_map(&mb, b, terms)) return cudaErrorInvalidValue;
  GemmParams p{};
  p.ep = ep;
  p.rows = (int)rows; p.cols = (int)cols; p.k = (int)k;
  p.tiles_m = g.tiles_m; p.tiles_n = g.tiles_n; p.splits = g.splits; p.kblocks = g.kblocks; p.per_split = g.per_split;
  p.a_mn = a.mn; p.b_mn = b.mn;
  auto even = [](const void* q, long long ld) { return !q || (ld % 2 == 0 && reinterpret_cast<uintptr_t>(q) % 4 == 0); };
  p.pairs = cols % 2 == 0 && even(ep.y, ep.ldy) && even(ep.z, ep.ldy) && even(ep.residual, ep.ldr);
  p.flags = flags;
  p.ep.parts = g.splits > 1 ? parts : nullptr;
  const bool turns = g.per_split > Gemm<1, 1>::kTurn;
  auto launch = terms == 3 ? (g.cg == 2 ? launch_gemm<2, 3, true> : launch_gemm<1, 3, true>)
                : turns    ? (g.cg == 2 ? launch_gemm<2, 1, true> : launch_gemm<1, 1, true>)
                           : (g.cg == 2 ? launch_gemm<2, 1, false> : launch_gemm<1, 1, false>);
  cudaError_t e = launch(ma, mb, p, st);
  if (e != cudaSuccess || g.splits == 1) return e;
  const int col_blocks = (int)((cols + 31) / 32);
  const unsigned grid = (unsigned)(col_blocks * ((rows + 63) / 64));
  return terms == 1 ? launch_pdl(linear_join_kernel<true>, grid, 256, 0, st, static_cast<const float*>(parts), g.splits, p.rows,
                                 p.cols, p.k, col_blocks, ep)
                    : launch_pdl(linear_join_kernel<false>, grid, 256, 0, st, static_cast<const float*>(parts), g.splits, p.rows,
                                 p.cols, p.k, col_blocks, ep);
}

// Where an operand's terms go, and whether it needs them at all.
bool direct(const gdn2_linear_desc* d, const void* p, long long ld) {
  return d->dtype == GDN2_BF16 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
long long padded(long long n) { return (n + 7) / 8 * 8; }
size_t terms_bytes(const gdn2_linear_desc* d, long long rows, long long cols) {
  return round256((size_t)rows * padded(cols) * 2 * (d->dtype == GDN2_F32 ? 3 : 1));
}
TermsJob terms_job(const void* p, long long ld, long long rows, long long cols, void* to) {
  const long long ldt = padded(cols);
  return {p, static_cast<__nv_bfloat16*>(to), ld, ldt, rows * (ldt / 8), (int)rows, (int)cols};
}
cudaError_t make_terms(const gdn2_linear_desc* d, const TermsJob& a, const TermsJob& b, cudaStream_t st) {
  const long long want = (a.items + b.items + 255) / 256;
  if (!want) return cudaSuccess;
  const unsigned grid = (unsigned)(want < kSMs * 32 ? want : kSMs * 32);
  if (d->dtype == GDN2_F32) linear_terms_kernel<float><<<grid, 256, 0, st>>>(a, b);
  else linear_terms_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, b);
  return cudaGetLastError();
}

gdn2_status check_linear(const gdn2_linear_desc* d) {
  if (!d || d->M < 0 || d->K < 1 || d->N < 1) return GDN2_ERR_INVALID_ARGUMENT;
  if ((d->dtype != GDN2_F32 && d->dtype != GDN2_BF16) || (d->bias_dtype != GDN2_F32 && d->bias_dtype != GDN2_BF16))
    return GDN2_ERR_INVALID_ARGUMENT;
  if (d->act != GDN2_ACT_NONE && d->act != GDN2_ACT_GELU_TANH) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->x_stride < d->K || d->w_stride < d->N || d->res_stride < 0) return GDN2_ERR_INVALID_ARGUMENT;
  if (d->M > 1 << 28 || d->K > 1 << 28 || d->N > 1 << 28) return GDN2_ERR_UNSUPPORTED;
  const long long most = 1ll << 36;     // strides and terms of a tensor map stay below 2^40 bytes
  if (d->x_stride > 1ll << 28 || d->w_stride > 1ll << 28 || (long long)d->M * d->N > most ||
      (long long)d->M * d->x_stride > most || (long long)d->K * d->w_stride > most)
    return GDN2_ERR_UNSUPPORTED;
  return GDN2_OK;
}
bool off(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
size_t element(const gdn2_linear_desc* d) { return d->dtype == GDN2_BF16 ? 2 : 4; }

// Rows that are multiplied without the tensor cores.  fp32: where W would first be cut into terms (8 x 512 x 4608 10.7 us
// against 16.3, 16 x 4096 x 4096 43 against about 50); bf16 rows are few where a launch less counts (4 x 512 x 4608 5.8 us
// against 8.1; of 8 rows 11.2 against 8.1, 8 x 4096 x 4096 21 against 15).
int few_rows(const gdn2_linear_desc* d) { return d->dtype == GDN2_F32 ? 16 : 4; }
// The small kernel takes about 2 + k / 64 us for a sum over k where every tile has an SM of its own, and all tiles' work
// shared out where they have not.  It is taken where that is less than the tiled path takes at such sizes: forward 11 to
// 15 us in fp32 (of which making the terms is 4) and 5 to 8 in bf16; dx with dW 19 to 32 and 12 to 24, one of them alone
// 10 to 18 and 4 to 5, with GELU's dz to make 6 to 12.  fp32 64 x 128 x 96 forward 10.5 -> 4.6 us, backward 19.8 -> 4.7; 128 x 512 x 256
// 13.6 -> 10.6 and 24.8 -> 9.0; 256 x 256 x 256 13.1 -> 6.6 and 29.2 -> 7.8; 128 x 1024 x 128 14.2 against 18.7: not taken.
// bf16 64 x 128 x 96 6.0 -> 4.6 and 13.0 -> 4.8; 128 x 512 x 256 8.1 against 11.2: not taken.
struct SmallSize { long long tiles, steps; };
SmallSize small_size(long long rows, long long cols, long long k) {
  return {(rows + kSmallTile - 1) / kSmallTile * ((cols + kSmallTile - 1) / kSmallTile), (k + kSmallK - 1) / kSmallK + 2};
}
bool small_within(SmallSize a, SmallSize b, int us) {
  const long long sms = kSMs, most = std::max(a.steps, b.steps);
  if (a.tiles + b.tiles <= sms) return most <= us;
  return a.tiles <= us * sms && b.tiles <= us * sms && 2 * (a.tiles * a.steps + b.tiles * b.steps) + most * sms <= 2 * us * sms;
}
bool small_fwd(const gdn2_linear_desc* d) {
  return small_within(small_size(d->M, d->N, d->K), {}, d->dtype == GDN2_F32 ? 11 : 6);
}
bool small_bwd(const gdn2_linear_desc* d, bool dx, bool dw, bool db) {
  if ((!dx && !dw) || (db && !dw)) return false;          // a sum of columns alone has no tiles here
  const bool f32 = d->dtype == GDN2_F32;
  return small_within(dx ? small_size(d->M, d->K, d->N) : SmallSize{}, dw ? small_size(d->K, d->N, d->M) : SmallSize{},
                      dx && dw ? (f32 ? 19 : 12) : f32 ? 11 : d->act != GDN2_ACT_NONE ? 7 : 4);
}
int small_tiles(const Product& p) { return (int)small_size(p.rows, p.cols, p.k).tiles; }
cudaError_t run_small(const gdn2_linear_desc* d, const Product& p0, const Product& p1, cudaStream_t st) {
  Products both{{p0, p1}, small_tiles(p0)};
  const int tiles = both.tiles0 + small_tiles(p1);
  if (d->dtype == GDN2_F32) linear_small_kernel<float><<<tiles, kSmallThreads, 0, st>>>(both);
  else linear_small_kernel<__nv_bfloat16><<<tiles, kSmallThreads, 0, st>>>(both);
  return cudaGetLastError();
}
struct FwdPlan {
  bool few, x_terms, w_terms;
  size_t x_at, w_at, parts_at, total;
};
FwdPlan plan_fwd(const gdn2_linear_desc* d, bool x_direct, bool w_direct) {
  FwdPlan f{};
  f.few = d->M <= few_rows(d);
  if (f.few || small_fwd(d)) return f;
  f.x_terms = !x_direct;
  f.w_terms = !w_direct;
  f.w_at = f.x_terms ? terms_bytes(d, d->M, d->K) : 0;
  f.parts_at = f.w_at + (f.w_terms ? terms_bytes(d, d->K, d->N) : 0);
  f.total = f.parts_at + parts_of(plan_gemm(d->M, d->N, d->K, d->dtype == GDN2_F32 ? 3 : 1), d->M, d->N);
  return f;
}

constexpr int kBand = 256;              // rows of a CTA of the dz kernel
struct BwdPlan {
  bool dz, x_terms, w_terms;            // dz: its own buffer (an activation, fp32, or rows not on 16 bytes)
  size_t dz_at, w_at, x_at, db_at, parts_at, total;
};
BwdPlan plan_bwd(const gdn2_linear_desc* d, bool dx, bool dw, bool db, bool x_direct, bool w_direct, bool dy_direct) {
  BwdPlan b{};
  if (small_bwd(d, dx, dw, db)) return b;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t r = at; at += round256(n); return r; };
  b.dz = (dx || dw) && (!dy_direct || d->act != GDN2_ACT_NONE);
  if (b.dz) b.dz_at = take(terms_bytes(d, d->M, d->N));
  b.w_terms = dx && !w_direct;
  b.x_terms = dw && !x_direct;
  if (b.w_terms) b.w_at = take(terms_bytes(d, d->K, d->N));
  if (b.x_terms) b.x_at = take(terms_bytes(d, d->M, d->K));
  if (db) b.db_at = take((size_t)((d->M + kBand - 1) / kBand) * d->N * 4);
  b.parts_at = at;
  size_t parts = 0;
  const int terms = d->dtype == GDN2_F32 ? 3 : 1;
  if (dx) parts = parts_of(plan_gemm(d->M, d->K, d->N, terms), d->M, d->K);
  if (dw) {
    const size_t q = parts_of(plan_gemm(d->K, d->N, d->M, terms), d->K, d->N);
    if (q > parts) parts = q;
  }
  b.total = at + parts;
  return b;
}

template <class T, int V>
cudaError_t launch_few(FewParams p, cudaStream_t st) {
  const long long blocks = (p.cols + 32 * V - 1) / (32 * V);
  p.clusters = 1;
  while (p.clusters < 8 && blocks * p.clusters < 2 * kSMs && p.k / p.clusters >= 64) p.clusters *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * p.clusters));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)p.clusters;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (p.rows == 1) return cudaLaunchKernelEx(&cfg, linear_few_kernel<T, V, 1>, p);
  if constexpr (sizeof(T) == 4)
    if (p.rows > 4) return cudaLaunchKernelEx(&cfg, linear_few_kernel<T, V, 8>, p);
  return cudaLaunchKernelEx(&cfg, linear_few_kernel<T, V, 4>, p);
}
// Four columns to a lane where that leaves a CTA for every SM.
template <class T>
cudaError_t launch_few(const FewParams& p, cudaStream_t st) {
  return (p.cols + 127) / 128 * 8 >= kSMs ? launch_few<T, 4>(p, st) : launch_few<T, 1>(p, st);
}
cudaError_t run_few(const gdn2_linear_desc* d, const FewParams& all, cudaStream_t st) {
  for (int r = 0; r < d->M; r += 8) {   // eight rows a launch
    FewParams p = all;
    const size_t el = element(d);
    p.rows = d->M - r < 8 ? d->M - r : 8;
    p.x = static_cast<const uint8_t*>(p.x) + (size_t)r * p.ldx * el;
    p.ep.y = static_cast<uint8_t*>(p.ep.y) + (size_t)r * p.ep.ldy * el;
    if (p.ep.z) p.ep.z = static_cast<uint8_t*>(p.ep.z) + (size_t)r * p.ep.ldy * el;
    if (p.ep.residual) p.ep.residual = static_cast<const uint8_t*>(p.ep.residual) + (size_t)r * p.ep.ldr * el;
    const cudaError_t e = d->dtype == GDN2_F32 ? launch_few<float>(p, st) : launch_few<__nv_bfloat16>(p, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace gdn2

extern "C" size_t gdn2_linear_fwd_workspace_bytes(const gdn2_linear_desc* d) {
  using namespace gdn2;
  if (check_linear(d) != GDN2_OK || !d->M) return 0;
  const bool bf16 = d->dtype == GDN2_BF16;
  return plan_fwd(d, bf16 && d->x_stride % 8 == 0, bf16 && d->w_stride % 8 == 0).total;
}

extern "C" gdn2_status gdn2_linear_fwd(const gdn2_linear_desc* d, const void* x, const void* w, const void* bias,
                                       const void* residual, void* y, void* z, void* workspace, uint32_t* flags,
                                       void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_linear(d);
  if (s != GDN2_OK) return s;
  if (!d->M) return GDN2_OK;
  const size_t el = element(d);
  if (!x || !w || !y || !flags || off(x, 16) || off(w, 16) || off(y, el) || off(z, el) || off(residual, el) ||
      off(bias, d->bias_dtype == GDN2_BF16 ? 2 : 4))
    return GDN2_ERR_INVALID_ARGUMENT;
  const FwdPlan f = plan_fwd(d, direct(d, x, d->x_stride), direct(d, w, d->w_stride));
  if (f.total && (!workspace || off(workspace, 256))) return GDN2_ERR_INVALID_ARGUMENT;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Epilogue ep{};
  ep.y = y; ep.z = z; ep.bias = bias; ep.residual = residual;
  ep.ldr = d->res_stride; ep.ldy = d->N;
  ep.y_bf16 = d->dtype == GDN2_BF16; ep.bias_bf16 = d->bias_dtype == GDN2_BF16; ep.act = d->act;
  cudaError_t e = cudaSuccess;
  if (f.few) {
    FewParams p{};
    p.ep = ep;
    p.x = x; p.w = w; p.ldx = d->x_stride; p.ldw = d->w_stride; p.cols = d->N; p.k = d->K;
    e = run_few(d, p, st);
  } else if (small_fwd(d)) {
    Product p{};
    p.a = x; p.a_row = d->x_stride; p.a_k = 1;
    p.b = w; p.b_k = d->w_stride; p.b_col = 1;
    p.rows = d->M; p.cols = d->N; p.k = d->K;
    p.ep = ep;
    e = run_small(d, p, Product{}, st);
  } else {
    const int terms = d->dtype == GDN2_F32 ? 3 : 1;
    if (terms == 3) {
      ep.a = static_cast<const float*>(x); ep.a_row = d->x_stride; ep.a_k = 1;
      ep.b = static_cast<const float*>(w); ep.b_col = 1; ep.b_k = d->w_stride;
    }
    Operand a{x, d->M, d->K, d->x_stride, 0, false}, b{w, d->K, d->N, d->w_stride, 0, true};
    TermsJob jx{}, jw{};
    if (f.x_terms) {
      jx = terms_job(x, d->x_stride, d->M, d->K, ws + f.x_at);
      a.p = ws + f.x_at; a.ld = padded(d->K); a.term = d->M * a.ld;
    }
    if (f.w_terms) {
      jw = terms_job(w, d->w_stride, d->K, d->N, ws + f.w_at);
      b.p = ws + f.w_at; b.ld = padded(d->N); b.term = d->K * b.ld;
    }
    e = make_terms(d, jx, jw, st);
    if (e == cudaSuccess)
      e = gemm(a, b, terms, ep, d->M, d->N, d->K, reinterpret_cast<float*>(ws + f.parts_at), flags, st);
  }
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}

extern "C" size_t gdn2_linear_bwd_workspace_bytes(const gdn2_linear_desc* d, int32_t want) {
  using namespace gdn2;
  if (check_linear(d) != GDN2_OK || !d->M) return 0;
  const bool bf16 = d->dtype == GDN2_BF16;
  return plan_bwd(d, want & 1, want & 2, want & 4, bf16 && d->x_stride % 8 == 0, bf16 && d->w_stride % 8 == 0,
                  bf16 && d->N % 8 == 0).total;
}

extern "C" gdn2_status gdn2_linear_bwd(const gdn2_linear_desc* d, const void* x, const void* w, const void* z,
                                       const void* dy, void* dx, void* dw, void* db, void* workspace, uint32_t* flags,
                                       void* stream) {
  using namespace gdn2;
  const gdn2_status s = check_linear(d);
  if (s != GDN2_OK) return s;
  const size_t el = element(d);
  if (d->M < 1 || !dy || !flags || (dx && !w) || (dw && !x) || (d->act != GDN2_ACT_NONE && !z) || off(x, 16) || off(w, 16) ||
      off(dy, 16) || off(z, el) || off(dx, el) || off(dw, el) || off(db, d->bias_dtype == GDN2_BF16 ? 2 : 4))
    return GDN2_ERR_INVALID_ARGUMENT;
  if (!dx && !dw && !db) return GDN2_OK;
  const BwdPlan b = plan_bwd(d, dx, dw, db, direct(d, x, d->x_stride), direct(d, w, d->w_stride), direct(d, dy, d->N));
  if (b.total && (!workspace || off(workspace, 256))) return GDN2_ERR_INVALID_ARGUMENT;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool act = d->act != GDN2_ACT_NONE, bf16 = d->dtype == GDN2_BF16;
  const int terms = bf16 ? 1 : 3, bands = (d->M + kBand - 1) / kBand;
  const long long ldz = padded(d->N);
  cudaError_t e = cudaSuccess;
  if (small_bwd(d, dx, dw, db)) {
    Product px{}, pw{};
    if (dx) {
      px.a = dy; px.z = act ? z : nullptr; px.a_row = d->N; px.a_k = 1;
      px.b = w; px.b_k = 1; px.b_col = d->w_stride;
      px.rows = d->M; px.cols = d->K; px.k = d->N;
      px.ep.y = dx; px.ep.ldy = d->K; px.ep.y_bf16 = bf16;
    }
    if (dw) {
      pw.a = x; pw.a_row = 1; pw.a_k = d->x_stride;
      pw.b = dy; pw.z = act ? z : nullptr; pw.z_of_b = 1; pw.b_k = d->N; pw.b_col = 1;
      pw.rows = d->K; pw.cols = d->N; pw.k = d->M;
      pw.ep.y = dw; pw.ep.ldy = d->N; pw.ep.y_bf16 = bf16;
      pw.sums = db; pw.sums_bf16 = d->bias_dtype == GDN2_BF16;
    }
    return run_small(d, px, pw, st) == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
  }
  if (b.dz || db) {
    const int col_blocks = (d->N + 63) / 64;
    const unsigned grid = (unsigned)(col_blocks * (long long)bands);
    __nv_bfloat16* out = b.dz ? reinterpret_cast<__nv_bfloat16*>(ws + b.dz_at) : nullptr;
    float* parts = db ? reinterpret_cast<float*>(ws + b.db_at) : nullptr;
    auto go = [&](auto kernel, auto t) {
      using T = decltype(t);
      kernel<<<grid, 256, 0, st>>>(static_cast<const T*>(dy), static_cast<const T*>(z), d->M, d->N, kBand, col_blocks, out, ldz,
                                   parts);
    };
    if (bf16) act ? go(linear_dz_kernel<__nv_bfloat16, true>, __nv_bfloat16()) : go(linear_dz_kernel<__nv_bfloat16, false>, __nv_bfloat16());
    else act ? go(linear_dz_kernel<float, true>, 0.f) : go(linear_dz_kernel<float, false>, 0.f);
    e = cudaGetLastError();
    if (db && e == cudaSuccess) {
      e = launch_pdl(linear_db_kernel, (unsigned)((d->N + 31) / 32), 256, 0, st, static_cast<const float*>(parts), bands, d->N, db,
                     (int)(d->bias_dtype == GDN2_BF16));
    }
  }
  const void* pz = b.dz ? static_cast<const void*>(ws + b.dz_at) : dy;
  const long long ldp = b.dz ? ldz : d->N, term_z = d->M * ldz;
  const float* dz_plain = bf16 ? nullptr : static_cast<const float*>(dy);
  const float* z_plain = bf16 || !act ? nullptr : static_cast<const float*>(z);
  float* parts = reinterpret_cast<float*>(ws + b.parts_at);
  if (e == cudaSuccess)
    e = make_terms(d, b.x_terms ? terms_job(x, d->x_stride, d->M, d->K, ws + b.x_at) : TermsJob{},
                   b.w_terms ? terms_job(w, d->w_stride, d->K, d->N, ws + b.w_at) : TermsJob{}, st);
  if (dx && e == cudaSuccess) {
    Operand bo{w, d->K, d->N, d->w_stride, 0, false};
    if (b.w_terms) {
      bo.p = ws + b.w_at; bo.ld = padded(d->N); bo.term = d->K * bo.ld;
    }
    Epilogue ep{};
    ep.y = dx; ep.ldy = d->K; ep.y_bf16 = bf16;
    if (!bf16) {
      ep.a = dz_plain; ep.az = z_plain; ep.a_row = d->N; ep.a_k = 1;
      ep.b = static_cast<const float*>(w); ep.b_col = d->w_stride; ep.b_k = 1;
    }
    if (e == cudaSuccess) e = gemm({pz, d->M, d->N, ldp, term_z, false}, bo, terms, ep, d->M, d->K, d->N, parts, flags, st);
  }
  if (dw && e == cudaSuccess) {
    Operand a{x, d->M, d->K, d->x_stride, 0, true};
    if (b.x_terms) {
      a.p = ws + b.x_at; a.ld = padded(d->K); a.term = d->M * a.ld;
    }
    Epilogue ep{};
    ep.y = dw; ep.ldy = d->N; ep.y_bf16 = bf16;
    if (!bf16) {
      ep.a = static_cast<const float*>(x); ep.a_row = 1; ep.a_k = d->x_stride;
      ep.b = dz_plain; ep.bz = z_plain; ep.b_col = 1; ep.b_k = d->N;
    }
    if (e == cudaSuccess) e = gemm(a, {pz, d->M, d->N, ldp, term_z, true}, terms, ep, d->K, d->N, d->M, parts, flags, st);
  }
  return e == cudaSuccess ? GDN2_OK : GDN2_ERR_CUDA;
}
