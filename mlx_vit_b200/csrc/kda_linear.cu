// Linear products with a fused epilogue, on the 5th-generation tensor cores (16-bit operands,
// float32 accumulation in tensor memory):
//
//   forward   y  = act(x W^T + bias) + residual, and z = x W^T + bias kept for the backward
//   dgrad     dx = dz W,  or  (dz W) * act'(z) where an activation lies below
//   wgrad     dW = dz^T x
//
// and db, the column sums of dz, from the pass that makes dz (dgrad's epilogue, or the activation-gradient
// pass).  (A product of dz^T with ones beside dW summed them without another pass, but each change
// between the two accumulators cost the tensor cores some 100 ns: 90 us against 76 for dW of 4096 x 1024.)
//
// One kernel: C[m][n] = sum_k A[m][k] B[n][k] over tiles of 128 CG x BN, where each operand lies in
// memory k-contiguous ("K-major") or m- / n-contiguous ("MN-major": the transposes are read in
// place).  Each persistent CTA (or pair of CTAs, CG = 2, whose tensor cores work on one tile and read
// half of B each) walks its tiles with one thread copying operand blocks of 64 k by TMA into a
// ring of stages, one thread issuing the products, and sixteen warps taking finished accumulators
// from tensor memory through the epilogue while the next tile's products run (two accumulators).
// Rows, columns and k past the end are TMA's zero fill and clipped stores.  Where the tiles are too few
// to fill the GPU, k is split: each part writes its float32 tile to a workspace and a second kernel
// adds the parts in order and runs the epilogue.  The tensor cores' operands have 16 bits, so what is computed
// here and multiplied again (an MLP's hidden activation, the gradient at z) is rounded to them once, and z is
// kept in them: a layer's gradients behind an activation are off by 2.4e-3 (bf16, 2-norm) where their own rounding
// makes 1.7e-3; carrying a second operand of the remainders would double the backward's products.  Sums (accumulators,
// parts, column sums) are float32 throughout.  A few rows (M <= 16, <= 32 of fewer outputs) take a kernel of their own
// that streams the weights once through registers.
//
// Bound by the tensor cores where the tiles fill the GPU: 4096 x 2048 x 8192 in bf16 92-98 us (1400-1490
// TFLOP/s, tensor pipe 80 % active), 12544 x 4096 x 1024 80 us, 8192^3 727 us (1510); in long runs by the
// power limit.  Small products are latency: 4.2 us for one block of k, 0.23 us for each block more.
#include <limits.h>

#include <atomic>
#include <initializer_list>

#include "kda_act.cuh"
#include "kda_common.cuh"
#include "kda_mma.cuh"
#include "kda_tc05.cuh"
#include "kda_tma.cuh"

namespace kda {
namespace linear {

// set to a KDA_ERR_* code by a bounded wait that gave up (read by kda_device_status)
static __device__ int g_linear_status;

constexpr int kThreads = 640;     // producer, issuer, allocator, idle, 16 epilogue warps
constexpr int kEpiWarp = 4, kEpiWarps = 16;
constexpr int kBlockK = 64;       // k per stage: 128 bytes, the swizzle's width
constexpr int kStageA = 128 * 128;
constexpr int kStaging = kEpiWarps * 4096;  // a 32 x 64 tile a warp
constexpr int kSmemMax = 232448;
constexpr int kPolls = 1 << 20;   // bound of a wait: some tens of milliseconds and more, against microseconds of work

enum { kInNone = 0, kInAdd = 1, kInActGrad = 2 };

struct alignas(64) Args {
  CUtensorMap a, b, out, in, z;   // split: out is the workspace of partial tiles
  int64_t ldo, ldi, ldz, ldp;
  const void *bias, *in_ptr;
  void *out_ptr, *z_ptr;
  float *part;          // split: [splits][tiles_m 128 CG][ldp] partial products
  float *sums;          // [32-row groups][n] column sums of what the epilogue writes, or null
  int m, n, k, tiles_m, tiles_n, splits, per_split;  // per_split: blocks of 64 k a part takes
  uint32_t idesc;
  int act, in_kind, out_tma, in_tma, save_z;
};

template <int CG, int BN>
struct Shape {
  static constexpr int kStageB = BN / CG * 128;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kFixed = kStaging + kEpiWarps * 128 + 512;
  static constexpr int kStages = (kSmemMax - kFixed) / kStage < 8 ? (kSmemMax - kFixed) / kStage : 8;
  static constexpr int kBufs = 2;           // accumulators of BN tensor-memory columns
  static constexpr int kCols = kBufs * BN;  // 128, 256 or 512: a power of two, as allocations are
  static constexpr int kSmem = kStages * kStage + kFixed;
};

// ---- what pairs of CTAs need ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {  // addr: a shared::cluster address
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" :: "r"(addr) : "memory");
}
__device__ __forceinline__ bool wait(uint32_t mbar, uint32_t parity, int polls = kPolls) {
  return mbar_wait(mbar, parity, polls);
}
// by a whole warp, with one answer for it: a warp that elects threads must not part
__device__ __forceinline__ bool wait_warp(uint32_t mbar, uint32_t parity) {
  return __all_sync(0xFFFFFFFFu, wait(mbar, parity));
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t mbar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n"
        :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(mbar) : "memory");
  else  // the barrier is the pair's first CTA's
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n"
        :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(mbar) : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap *map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];\n"
               :: "l"(map), "r"(src), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];\n" :: "l"(map) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;\n" :: "n"(N) : "memory"); }

// One thread of a converged warp.  The copying and the issuing warp run their loops whole and elect a
// thread for each instruction: its operands stay warp-uniform, in uniform registers.  (A loop
// inside `if (lane == 0)` moved every operand there first: 0.33 us for a block of 64 k at the least,
// whatever the tile.)
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// The low words of umma_desc(): start address and leading offset; kDescHigh: stride 1024, version,
// 128-byte swizzle.  A K step is 32 bytes further (K-major) or 16 rows (MN-major).
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
template <bool MN>
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr) { return (saddr >> 4) | ((MN ? 8192u >> 4 : 1u) << 16); }
template <bool MN>
constexpr uint32_t kDescStep = MN ? 2048 >> 4 : 32 >> 4;

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n"
        :: "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh) : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n}\n"
        :: "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t mbar) {  // to the barrier at this offset in every CTA of the pair
  if constexpr (CG == 1) tc_commit(mbar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
        :: "r"(mbar), "h"((uint16_t)3) : "memory");
}
template <int CG>
__device__ __forceinline__ void alloc(uint32_t dst, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" :: "r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" :: "r"(taddr), "r"(cols) : "memory");
}

// byte offset of 16-byte chunk c of row r in a tile of 128-byte rows with the 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// pack_z: of a pre-activation, whose value past the type's range, finite as it may be in float32, becomes the type's
// largest: every derivative has its limit there, and 0 times infinity at the infinity itself.  A NaN stays one.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const type v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ uint32_t pack_z(float a, float b) {
    uint32_t u;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
    return u;
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
};
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const type v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ uint32_t pack_z(float a, float b) {
    uint32_t u;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
    return u;
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const type *>(&u)); }
};

template <typename T>
__device__ __forceinline__ void store_z(T *p, float v) {
  const unsigned short u = (unsigned short)Pair<T>::pack_z(v, 0.f);
  *p = *reinterpret_cast<const T *>(&u);
}

// A 32 x 64 tile between global memory and a warp's staging rows where no TMA map can describe the
// matrix (a row pitch or a base that 16 bytes do not divide): coalesced 2-byte accesses.
template <typename T>
__device__ __forceinline__ void tile_in(uint8_t *st, const T *p, int64_t ld, int rows, int cols, int lane) {
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 8) {
    T v[8][2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + (i >> 1), c = lane + 32 * (i & 1);
      v[i >> 1][i & 1] = r < rows && c < cols ? p[r * ld + c] : T(0.f);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + (i >> 1), c = lane + 32 * (i & 1);
      *reinterpret_cast<T *>(st + chunk_at(r, c >> 3) + (c & 7) * 2) = v[i >> 1][i & 1];
    }
  }
}
template <typename T>
__device__ __forceinline__ void tile_out(const uint8_t *st, T *p, int64_t ld, int rows, int cols, int lane) {
  for (int r = 0; r < rows; ++r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = lane + 32 * h;
      if (c < cols) p[r * ld + c] = *reinterpret_cast<const T *>(st + chunk_at(r, c >> 3) + (c & 7) * 2);
    }
  }
}

// One 32 x 64 chunk of an accumulator to a warp's staging rows: bias, the activation (kForward) or
// its derivative at the staged z (kGrad), the staged residual, and z itself.
enum { kPlain = 0, kForward = 1, kGrad = 2 };
template <typename T, int KIND, int ACT>
__device__ __forceinline__ void finish8(float (&v)[8], uint4 *slot, bool add) {
  using P = Pair<T>;
  if (KIND == kGrad && ACT != KDA_ACT_NONE) {
    const uint4 zi = *slot;
    const uint32_t w[4] = {zi.x, zi.y, zi.z, zi.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 d = grad_through2(ACT, make_float2(v[2 * j], v[2 * j + 1]), P::unpack(w[j]));
      v[2 * j] = d.x;
      v[2 * j + 1] = d.y;
    }
  } else if (KIND == kForward) {
    if (ACT != KDA_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = activate2(ACT, make_float2(v[2 * j], v[2 * j + 1]));
        v[2 * j] = a.x;
        v[2 * j + 1] = a.y;
      }
    }
    if (add) {
      const uint4 ri = *slot;
      const uint32_t w[4] = {ri.x, ri.y, ri.z, ri.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = P::unpack(w[j]);
        v[2 * j] += x.x;
        v[2 * j + 1] += x.y;
      }
    }
  }
}
// Column lane % 8 of eight columns' sums over the warp's lanes: halves are exchanged while columns are
// left, then the four groups of lanes are added.
__device__ __forceinline__ float column_sum(const float (&v)[8], int lane) {
  float a[4], b[2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = (lane & 4 ? v[i + 4] : v[i]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 4 ? v[i] : v[i + 4], 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = (lane & 2 ? a[i + 2] : a[i]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 2 ? a[i] : a[i + 2], 2);
  float s = (lane & 1 ? b[1] : b[0]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 1 ? b[0] : b[1], 1);
  s += __shfl_xor_sync(0xFFFFFFFFu, s, 8);
  return s + __shfl_xor_sync(0xFFFFFFFFu, s, 16);
}
// `keep`: the accumulator with its bias as it is (z), else finished.  bs: the chunk's bias.  sums (kGrad, or
// null): where the column sums of the warp's `rows` rows go, before they are rounded.
template <typename T, int KIND, int ACT>
__device__ __forceinline__ void chunk(const Args &g, uint32_t acc, uint8_t *so, const T *bs, int lane, bool keep,
                                      float *sums = nullptr, int rows = 0, int cols = 0) {
  using P = Pair<T>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r[32];
    tmem_ld32(acc + 32 * h, r);
    tmem_wait_ld();
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // 8 columns: one 16-byte chunk of the row
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[8 * u + j]);
      if (KIND == kForward && g.bias) {
        const uint4 bi = *reinterpret_cast<const uint4 *>(bs + 32 * h + 8 * u);
        const uint32_t w[4] = {bi.x, bi.y, bi.z, bi.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = add2(make_float2(v[2 * j], v[2 * j + 1]), P::unpack(w[j]));
          v[2 * j] = x.x;
          v[2 * j + 1] = x.y;
        }
      }
      uint4 *slot = reinterpret_cast<uint4 *>(so + chunk_at(lane, 4 * h + u));
      if (!keep) finish8<T, KIND, ACT>(v, slot, g.in_kind == kInAdd);
      if (KIND == kGrad && sums) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = lane < rows ? v[j] : 0.f;
        const float s = column_sum(w, lane);
        const int j = 32 * h + 8 * u + lane;
        if (lane < 8 && j < cols) sums[j] = s;
      }
      *slot = keep ? make_uint4(P::pack_z(v[0], v[1]), P::pack_z(v[2], v[3]), P::pack_z(v[4], v[5]), P::pack_z(v[6], v[7]))
                   : make_uint4(P::pack(v[0], v[1]), P::pack(v[2], v[3]), P::pack(v[4], v[5]), P::pack(v[6], v[7]));
    }
  }
}

// Tile t's place: groups of kGroup rows of tiles, column by column, so that the CTAs at work at one time
// read few distinct rows of either operand.
constexpr int kGroup = 8;
__device__ __forceinline__ int2 place(int t, int tiles_m, int tiles_n) {
  const int group = t / (kGroup * tiles_n), in = t - group * kGroup * tiles_n, rows = min(kGroup, tiles_m - group * kGroup);
  return make_int2(group * kGroup + in % rows, in / rows);
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Args g) {
  using S = Shape<CG, BN>;
  extern __shared__ __align__(1024) uint8_t sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const uint32_t base = smem_u32(sm);
  if (base & 1023) {  // the swizzled tiles need a 1024-byte aligned base (every CTA has the same)
    if (tid == 0) atomicExch(&g_linear_status, KDA_ERR_MISALIGNED);
    return;
  }
  uint8_t *staging = sm + S::kStages * S::kStage;
  T *bias_sm = reinterpret_cast<T *>(staging + kStaging);
  // barriers: full[stages], empty[stages], acc_full[2], acc_empty[2], in[epilogue warps], idle; then tensor memory's address
  const uint32_t bars = smem_u32(bias_sm) + kEpiWarps * 128;
  const uint32_t full = bars, empty = full + 8 * S::kStages, acc_full = empty + 8 * S::kStages,
                 acc_empty = acc_full + 16, in_bar = acc_empty + 16, idle = in_bar + 8 * kEpiWarps, tmem_at = idle + 8;
  const int kblocks = (g.k + kBlockK - 1) / kBlockK;
  const int tiles = g.tiles_m * g.tiles_n, units = tiles * g.splits, first = blockIdx.x / CG, step = gridDim.x / CG;

  if (tid == 96) {  // the tensor maps on their way while barriers and tensor memory are set up (0.2 us of a small product)
    prefetch_map(&g.a);
    prefetch_map(&g.b);
    if (g.out_tma || g.splits > 1) prefetch_map(&g.out);
    if (g.in_kind && g.in_tma) prefetch_map(&g.in);
    if (g.save_z) prefetch_map(&g.z);
  }
  if (tid == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, kEpiWarps * CG);
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(in_bar + 8 * w, 1);
    mbar_init(idle, 1);
    mbar_fence_init();
  }
  if (warp == 2) alloc<CG>(tmem_at, S::kCols);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + (tmem_at - base));
  bool ok = true;

  if (warp == 0) {
    // ---- operand copies; both CTAs' bytes of a stage arrive on the first CTA's barrier ----
    const uint32_t full_lead = CG == 2 ? map_rank(full, 0) : full;
    uint32_t s = 0, ph = 1, issued = 0;
    for (int u = first; ok && u < units; u += step) {
      const int t = u % tiles, kb0 = u / tiles * g.per_split, kb1 = min(kblocks, kb0 + g.per_split);
      const int2 at_tile = place(t, g.tiles_m, g.tiles_n);
      const int m0 = at_tile.x * 128 * CG + (int)rank * 128, n0 = at_tile.y * BN + (int)rank * (BN / CG);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = wait_warp(empty + 8 * s, ph))) break;
        const uint32_t at = base + s * S::kStage, bt = at + kStageA, fb = full_lead + 8 * s;
        if (elect()) {
          if (rank == 0) mbar_expect_tx(full + 8 * s, S::kStage * CG);
          if (A_MN) {
            load_box<CG>(at, &g.a, m0, kb * kBlockK, fb);
            load_box<CG>(at + 8192, &g.a, m0 + 64, kb * kBlockK, fb);
          } else {
            load_box<CG>(at, &g.a, kb * kBlockK, m0, fb);
          }
          if (B_MN) {
#pragma unroll
            for (int j = 0; j < BN / CG / 64; ++j)
              load_box<CG>(bt + 8192 * j, &g.b, n0 + 64 * j, kb * kBlockK, fb);
          } else {
            load_box<CG>(bt, &g.b, kb * kBlockK, n0, fb);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == S::kStages) s = 0, ph ^= 1;
      }
    }
    if (!ok && rank == 0)  // gave up: let the copies in flight land before the CTA ends
      for (uint32_t i = issued > S::kStages ? issued - S::kStages : 0; i < issued; ++i)
        mbar_wait(full + 8 * (i % S::kStages), (i / S::kStages) & 1, 1 << 16);
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- products ----
      const uint32_t a_low = desc_low<A_MN>(base), b_low = desc_low<B_MN>(base + kStageA);
      uint32_t s = 0, ph = 0, n = 0;
      for (int u = first; ok && u < units; u += step, ++n) {
        const int kb0 = u / tiles * g.per_split, kb1 = min(kblocks, kb0 + g.per_split);
        const uint32_t buf = n % S::kBufs, use = n / S::kBufs;
        const uint32_t d = tmem + buf * BN;
        if (!(ok = wait_warp(acc_empty + 8 * buf, (use & 1) ^ 1))) break;
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_warp(full + 8 * s, ph))) break;
          tc_fence_after();
          const uint32_t al = a_low + s * (S::kStage >> 4), bl = b_low + s * (S::kStage >> 4);
          if (elect()) {
#pragma unroll
            for (int k = 0; k < kBlockK / 16; ++k)
              mma<CG>(d, al + k * kDescStep<A_MN>, bl + k * kDescStep<B_MN>, g.idesc, kb > kb0 || k > 0);
            commit<CG>(empty + 8 * s);
            if (kb + 1 == kb1) commit<CG>(acc_full + 8 * buf);
          }
          __syncwarp();
          if (++s == S::kStages) s = 0, ph ^= 1;
        }
      }
      if (!ok) {  // gave up: let the products in flight end before tensor memory is freed
        if (elect()) commit<CG>(idle);
        __syncwarp();
        mbar_wait(idle, 0, 1 << 16);
      }
    }
  } else if (warp >= kEpiWarp) {
    // ---- epilogue: warp (q, c) takes rows 32 q .. 32 q + 31 of the tile's 64-column chunk c.  Sixteen
    // warps, so that each scheduler has four to hide an accumulator's and a store's latency with ----
    const int e = warp - kEpiWarp, q = warp & 3, c = e >> 2;
    uint8_t *st = staging + e * 4096;
    const uint32_t st_at = smem_u32(st), my_in = in_bar + 8 * e;
    T *bs = bias_sm + e * 64;
    const uint32_t empty_lead = CG == 2 ? map_rank(acc_empty, 0) : acc_empty;
    uint32_t n = 0, in_phase = 0;
    // an accumulator's wait spans its whole sum: at least a microsecond's polls for each block of it
    const int acc_polls = (int)min((int64_t)INT_MAX, (int64_t)kPolls + 128 * (int64_t)g.per_split);
    const bool in_tma = g.in_kind && g.in_tma && g.splits == 1, ahead = in_tma && !g.save_z;
    for (int u = first; ok && u < units; u += step, ++n) {
      const int t = u % tiles, part = u / tiles;
      const uint32_t buf = n % S::kBufs, use = n / S::kBufs;
      const int2 at_tile = place(t, g.tiles_m, g.tiles_n);
      const int row0 = at_tile.x * 128 * CG + (int)rank * 128 + 32 * q, col0 = at_tile.y * BN + 64 * c;
      const bool mine = c < BN / 64 && row0 < g.m && col0 < g.n;
      const int rows = min(32, g.m - row0), cols = min(64, g.n - col0);
      auto fetch = [&] {  // residual or z into the staging tile (one lane)
        fence_proxy_async_smem();
        mbar_expect_tx(my_in, 4096);
        load_box<1>(st_at, &g.in, col0, row0, my_in);
      };
      // ahead of the accumulator: the staging tile's last store has been read, its next input, the bias
      if (lane == 0) store_wait_read<0>();
      __syncwarp();
      if (ahead && mine && lane == 0) fetch();
      if (g.bias && mine && g.splits == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = lane + 32 * h;
          bs[j] = j < cols ? static_cast<const T *>(g.bias)[col0 + j] : T(0.f);
        }
        __syncwarp();
      }
      if (lane == 0) ok = wait(acc_full + 8 * buf, use & 1, acc_polls);
      __syncwarp();
      if (!__all_sync(0xFFFFFFFFu, ok)) {
        ok = false;
        if (ahead && mine) mbar_wait(my_in, in_phase, 1 << 16);  // gave up: let the copy in flight land
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(32 * q) << 16);
      if (mine && g.splits > 1) {  // the float32 tile as it is, 32 columns a store
        const int prow = part * g.tiles_m * 128 * CG + row0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tmem_ld32(acc + 64 * c + 32 * h, r);
          if (h && lane == 0) store_wait_read<0>();
          __syncwarp();
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4 *>(st + chunk_at(lane, j)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            store_box(&g.out, st_at, col0 + 32 * h, prow);
            store_commit();
          }
        }
      } else if (mine) {
        if (g.save_z) {
          chunk<T, B_MN ? kPlain : kForward, KDA_ACT_NONE>(g, acc + 64 * c, st, bs, lane, true);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            store_box(&g.z, st_at, col0, row0);
            store_commit();
            store_wait_read<0>();
            if (in_tma) fetch();
          }
          __syncwarp();
        }
        if (in_tma) {
          ok = wait(my_in, in_phase);
          in_phase ^= 1;
          if (!__all_sync(0xFFFFFFFFu, ok)) {
            ok = false;
            break;
          }
        } else if (g.in_kind) {
          tile_in<T>(st, static_cast<const T *>(g.in_ptr) + row0 * g.ldi + col0, g.ldi, rows, cols, lane);
          __syncwarp();
        }
        if constexpr (A_MN) {
          chunk<T, kPlain, KDA_ACT_NONE>(g, acc + 64 * c, st, bs, lane, false);
        } else {
          constexpr int kind = B_MN ? kGrad : kForward;
          float *sums = B_MN && g.sums ? g.sums + (int64_t)(row0 >> 5) * g.n + col0 : nullptr;
          const uint32_t from = acc + 64 * c;
          switch (g.act) {
            case KDA_ACT_RELU: chunk<T, kind, KDA_ACT_RELU>(g, from, st, bs, lane, false, sums, rows, cols); break;
            case KDA_ACT_SILU: chunk<T, kind, KDA_ACT_SILU>(g, from, st, bs, lane, false, sums, rows, cols); break;
            case KDA_ACT_GELU: chunk<T, kind, KDA_ACT_GELU>(g, from, st, bs, lane, false, sums, rows, cols); break;
            case KDA_ACT_GELU_TANH: chunk<T, kind, KDA_ACT_GELU_TANH>(g, from, st, bs, lane, false, sums, rows, cols); break;
            default: chunk<T, kind, KDA_ACT_NONE>(g, from, st, bs, lane, false, sums, rows, cols);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (g.out_tma) {
          if (lane == 0) {
            store_box(&g.out, st_at, col0, row0);
            store_commit();
          }
        } else {
          tile_out<T>(st, static_cast<T *>(g.out_ptr) + row0 * g.ldo + col0, g.ldo, rows, cols, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) arrive_cluster(empty_lead + 8 * buf);
        else mbar_arrive(acc_empty + 8 * buf);
      }
    }
    if (lane == 0) store_wait_read<0>();
    __syncwarp();
  }
  if (!ok) atomicExch(&g_linear_status, KDA_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // neither CTA ends while the other's products or copies may touch it
  tc_fence_after();
  if (warp == 2) dealloc<CG>(tmem, S::kCols);
}

// Adds the parts of a split product in their order and runs the epilogue (its bytes, mostly out of the
// second-level cache: two parts of 2304 x 768 in 5.7 us), with SUMS on 32 rows a block
// whose column sums are its row of partials.
constexpr int kJoinRows = 4;  // rows a block of 64 x 4 threads takes at once; a thread takes 8 columns
template <typename T, bool SUMS>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args g, int64_t part_rows, int col_blocks) {
  using P = Pair<T>;
  constexpr int kRows = SUMS ? 32 : kJoinRows;
  const int64_t blk = blockIdx.x, row0 = blk / col_blocks * kRows;
  const int col = (int)(blk % col_blocks) * 512 + threadIdx.x * 8, k = min(8, g.n - col);
  float sum[8] = {};
  for (int64_t row = row0 + threadIdx.y; k > 0 && row < min(row0 + kRows, (int64_t)g.m); row += kJoinRows) {
    float v[8] = {};
    for (int p = 0; p < g.splits; ++p) {  // whole vectors: the workspace's columns are padded to tiles
      const float4 *src = reinterpret_cast<const float4 *>(g.part + (p * part_rows + row) * g.ldp + col);
      const float4 a = src[0], b = src[1];
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
    if (g.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < k) v[j] += to_f<T>(static_cast<const T *>(g.bias)[col + j]);
    }
    if (g.save_z) {
      T *z = static_cast<T *>(g.z_ptr) + row * g.ldz + col;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < k) store_z<T>(z + j, v[j]);
    }
    float x[8];
    if (g.in_kind) {
      const T *in = static_cast<const T *>(g.in_ptr) + row * g.ldi + col;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = j < k ? to_f<T>(in[j]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (g.in_kind == kInActGrad) v[j] = grad_through(g.act, v[j], x[j]);
      else v[j] = activate(g.act, v[j]) + (g.in_kind == kInAdd ? x[j] : 0.f);
      if (SUMS) sum[j] += v[j];
    }
    T *out = static_cast<T *>(g.out_ptr) + row * g.ldo + col;
    if (k == 8 && g.out_tma) {
      *reinterpret_cast<uint4 *>(out) = make_uint4(P::pack(v[0], v[1]), P::pack(v[2], v[3]), P::pack(v[4], v[5]), P::pack(v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < k) out[j] = from_f<T>(v[j]);
    }
  }
  if (SUMS) {
    __shared__ float red[kJoinRows][512 + 8];
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.y][threadIdx.x * 8 + j] = sum[j];
    __syncthreads();
    for (int t = threadIdx.y * 64 + threadIdx.x; t < 512; t += 256) {
      const int c = (int)(blk % col_blocks) * 512 + t;
      if (c < g.n) g.sums[(row0 >> 5) * g.n + c] = red[0][t] + red[1][t] + red[2][t] + red[3][t];
    }
  }
}

// ---- a few rows: y = act(x W^T + bias) + residual with M <= 32 ----
// The weights' bytes bound it: each is read once, straight into the fragments of m16n8k16 products
// whose 16 rows are rows of x and whose 8 columns are 8 outputs.  k may be summed in any order, so a
// lane's share of two products is 8 consecutive k (one 16-byte load of W, one of each row of x)
// instead of the layout's pairs.  `kw` warps share 8 or 16 outputs, each with its range of k, and the next eight
// loads of W a lane (4 KB a warp) are in flight while the last eight are multiplied; x comes
// through the first-level cache, which W's loads pass by.  The warps' sums meet in shared memory.
// Measured from memory, a call in a graph: 1 x 8192 x 2048 7.9 us (4.2 TB/s), 16 rows 9.8 us, 1 x 768 x 768
// 3.4 us, 1 x 50000 x 1024 21.3 us (4.8 TB/s).  Bound by the loads in flight while a wave starts and ends.
template <typename T>
__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes of a row of W, which no one reads again, and of x, which every warp reads.
__device__ __forceinline__ uint4 load_once(const char *p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
// `left` elements of 8 exist (none, if not positive); the others count as zero.  The load itself is
// a whole aligned 16 bytes, whose first byte lies in the row, so it stays in its page.
__device__ __forceinline__ uint4 load_some(const char *p, int left) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if (left > 0) u = __ldg(reinterpret_cast<const uint4 *>(p));
  if (left < 8) {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] &= left > 2 * j + 1 ? 0xFFFFFFFFu : left > 2 * j ? 0xFFFFu : 0u;
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return u;
}
struct FewArgs {
  const void *x, *w, *bias, *res;
  void *y, *z;
  int64_t ldx, ldw, ldr, ldy, ldz;
  int m, n, k, act;
};
constexpr int kFewRows = 32, kFewWarps = 8;
// With more than 16 rows x's way through the first-level cache bounds it; from 64 outputs an SM on the tiled kernel's
// tile for each is as fast or faster: 32 x 11008 x 4096 32.8 us here, 27.0 in tiles, 32 x 20000 x 512 18.3 and
// 11.5, 32 x 9473 x 2048 (one tile more than SMs) 19.7 and 18.8, 17 rows 17.9 and 21.5
static bool is_few(int64_t m, int64_t n, int sms) { return m <= 16 || (m <= kFewRows && n <= 64ll * sms); }
// MT groups of 8 rows of x (1, 2 or 4) by NB groups of 8 outputs a warp; with two a load of x serves two products
template <typename T, int MT, int NB>
__global__ void __launch_bounds__(32 * kFewWarps, 2) few_rows_kernel(const FewArgs a, int kw, int range) {
  __shared__ float red[kFewWarps][8 * MT][8 * NB + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int blocks = kFewWarps / kw, block0 = blockIdx.x * blocks;  // groups of 8 NB outputs of this CTA
  const int n0 = (block0 + warp / kw) * 8 * NB, from = warp % kw * range, to = min(from + range, a.k);
  const char *wr[NB], *xr[MT];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    wr[b] = static_cast<const char *>(a.w) + 2 * (a.ldw * min(n0 + 8 * b + g, a.n - 1) + from + 8 * c);
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = static_cast<const char *>(a.x) + 2 * (a.ldx * min(8 * t + g, a.m - 1) + from + 8 * c);
  constexpr int U = 8 / NB, P = (MT + 1) / 2;
  float d[NB][P][4] = {};
  auto products = [&](const uint4 (&w)[NB], const uint4 (&x)[2 * P]) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mma_m16n8k16<T>(d[b][p], x[2 * p].x, x[2 * p + 1].x, x[2 * p].y, x[2 * p + 1].y, w[b].x, w[b].y);
        mma_m16n8k16<T>(d[b][p], x[2 * p].z, x[2 * p + 1].z, x[2 * p].w, x[2 * p + 1].w, w[b].z, w[b].w);
      }
  };
  if (n0 < a.n) {
    const int whole = to > from ? (to - from) / (32 * U) : 0;
    uint4 next[U][NB];
    if (whole) {
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int b = 0; b < NB; ++b) next[j][b] = load_once(wr[b] + 64 * j);
    }
    for (int i = 0; i < whole; ++i) {
      uint4 w[U][NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int j = 0; j < U; ++j) w[j][b] = next[j][b];
        wr[b] += 64 * U;
      }
      if (i + 1 < whole) {
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int b = 0; b < NB; ++b) next[j][b] = load_once(wr[b] + 64 * j);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        uint4 x[2 * P];
#pragma unroll
        for (int t = 0; t < 2 * P; ++t)
          x[t] = t < MT ? __ldg(reinterpret_cast<const uint4 *>(xr[t < MT ? t : 0] + 64 * j)) : make_uint4(0, 0, 0, 0);
        products(w[j], x);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) xr[t] += 64 * U;
    }
    for (int k = from + 32 * U * whole + 8 * c; k - 8 * c < to; k += 32) {  // the range's rest
      uint4 w[NB], x[2 * P];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        w[b] = load_some(wr[b], to - k);
        wr[b] += 64;
      }
#pragma unroll
      for (int t = 0; t < 2 * P; ++t) {
        x[t] = t < MT ? load_some(xr[t < MT ? t : 0], to - k) : make_uint4(0, 0, 0, 0);
        if (t < MT) xr[t] += 64;
      }
      products(w, x);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * p + 8 * (i >> 1) < 8 * MT) red[warp][16 * p + g + 8 * (i >> 1)][8 * b + 2 * c + (i & 1)] = d[b][p][i];
  __syncthreads();
  const int outs = 8 * NB * blocks;
  for (int o = threadIdx.x; o < outs * a.m; o += 32 * kFewWarps) {
    const int j = o % outs, row = o / outs, n = 8 * NB * block0 + j;
    if (n >= a.n) continue;
    float v = 0.f;
    for (int i = 0; i < kw; ++i) v += red[j / (8 * NB) * kw + i][row][j % (8 * NB)];
    if (a.bias) v += to_f<T>(static_cast<const T *>(a.bias)[n]);
    if (a.z) store_z<T>(static_cast<T *>(a.z) + row * a.ldz + n, v);
    v = activate(a.act, v);
    if (a.res) v += to_f<T>(static_cast<const T *>(a.res)[row * a.ldr + n]);
    static_cast<T *>(a.y)[row * a.ldy + n] = from_f<T>(v);
  }
}

// dz = dy act'(z) over a [rows][cols] matrix (z null: a copy; dz null: none), any strides and alignments, and
// the column sums of dz.  A block takes 256 columns, 8 a thread (each matrix by 16 bytes where its
// rows allow it), of a range of rows, 8 at a time; its sums meet in shared memory and go to its row of
// partials.  Bound by its bytes: 12544 x 4096 with SiLU 54 us (5.7 TB/s), with the sums 57 and 3 to add them.
template <typename T, int ACT, bool SUMS>
__global__ void __launch_bounds__(256) act_grad_kernel(int64_t rows, int cols, const T *dy, int64_t ldy, const T *z, int64_t ldz,
                                                       T *dz, int64_t ldd, int vec_y, int vec_z, int vec_d, float *part, T *db) {
  using P = Pair<T>;
  auto unpack = [](const uint4 &u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = P::unpack(w[j]);
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  };
  const int c = blockIdx.x * 256 + threadIdx.x * 8, k = cols - c;
  float sum[8] = {};
  auto finish = [&](float (&x)[8], const float (&y)[8]) {
    if (ACT != KDA_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 d = grad_through2(ACT, make_float2(x[2 * j], x[2 * j + 1]), make_float2(y[2 * j], y[2 * j + 1]));
        x[2 * j] = d.x;
        x[2 * j + 1] = d.y;
      }
    }
    if (SUMS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += x[j];
    }
  };
  const int64_t step = (int64_t)gridDim.y * 8;
  int64_t r = (int64_t)blockIdx.y * 8 + threadIdx.y;
  if (k >= 8 && vec_y && (ACT == KDA_ACT_NONE || vec_z) && (!dz || vec_d)) {
    constexpr int R = 4;  // rows whose loads are in flight together
    for (; r < rows; r += R * step) {
      uint4 a[R], b[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (r + i * step >= rows) break;
        a[i] = *reinterpret_cast<const uint4 *>(dy + (r + i * step) * ldy + c);
        if (ACT != KDA_ACT_NONE) b[i] = *reinterpret_cast<const uint4 *>(z + (r + i * step) * ldz + c);
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (r + i * step >= rows) break;
        float x[8], y[8] = {};
        unpack(a[i], x);
        if (ACT != KDA_ACT_NONE) unpack(b[i], y);
        finish(x, y);
        if (dz)
          *reinterpret_cast<uint4 *>(dz + (r + i * step) * ldd + c) =
              make_uint4(P::pack(x[0], x[1]), P::pack(x[2], x[3]), P::pack(x[4], x[5]), P::pack(x[6], x[7]));
      }
    }
  } else if (k > 0) {
#pragma unroll 2
    for (; r < rows; r += step) {
      float x[8], y[8] = {};
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = j < k ? to_f<T>(dy[r * ldy + c + j]) : 0.f;
      if (ACT != KDA_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = j < k ? to_f<T>(z[r * ldz + c + j]) : 0.f;
      }
      finish(x, y);
      if (!dz) continue;
      T *out = dz + r * ldd + c;
      if (vec_d && k >= 8) {
        *reinterpret_cast<uint4 *>(out) = make_uint4(P::pack(x[0], x[1]), P::pack(x[2], x[3]), P::pack(x[4], x[5]), P::pack(x[6], x[7]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < k) out[j] = from_f<T>(x[j]);
      }
    }
  }
  if (SUMS) {
    __shared__ float red[8][256 + 8];
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.y][threadIdx.x * 8 + j] = sum[j];
    __syncthreads();
    const int t = threadIdx.y * 32 + threadIdx.x, col = blockIdx.x * 256 + t;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[i][t];
    if (col < cols) {
      if (gridDim.y == 1) db[col] = from_f<T>(v);  // no other partials
      else part[(int64_t)blockIdx.y * cols + col] = v;
    }
  }
}
// db[j] = sum over the partials, each thread row every 32nd of them, in their order
template <typename T>
__global__ void __launch_bounds__(1024) sums_kernel(const float *part, int parts, int cols, T *db) {
  __shared__ float red[32][33];
  const int j = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (j < cols) {
#pragma unroll 4
    for (int i = threadIdx.y; i < parts; i += 32) s += part[(int64_t)i * cols + j];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = red[threadIdx.x][threadIdx.y];  // column 32 block + y, its partial sum x
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < cols) db[col] = from_f<T>(s);
}

// ---- host side ----
static bool tma_able(const void *p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

static int device_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  static std::atomic<int> known[64];
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// ---- which tiles, and into how many parts k is split: the least estimated time.  A pair of CTAs on
// 256 x 256 moves the fewest bytes into shared memory for its products (64 KB for twice the work of
// four 128 x 128 tiles' 128 KB) and wins where its tiles fill the GPU (12544 x 2304 x 768 forward: 37 us,
// 49 on 128 x 128, 88 on 128 x 64); fewer rows or columns take smaller tiles (256 x 768 x 768: 10.4,
// 8.1 and 7.7 us), and long sums over few tiles are split (dW of 768 x 768 from 12544 rows: 61 us whole,
// 21 in eight parts; dW of 4096 x 1024, whose tiles nearly fill the GPU: 75 and 87 us in two) ----
struct Plan {
  int cg, bn, splits, per_split;
};
static Plan plan_for(int64_t m, int64_t n, int64_t k, int sms, bool may_split) {
  struct Tile {
    int cg, bn;
    double busy, alone;  // us a block of 64 k takes where the GPU is full, and on one tile alone (measured)
  };
  static const Tile tiles[] = {{2, 256, 0.40, 0.31}, {1, 128, 0.40, 0.26}, {1, 64, 0.31, 0.23}};
  const int64_t blocks = (k + kBlockK - 1) / kBlockK;
  Plan best = {};
  double best_us = 1e300;
  for (const Tile &t : tiles) {
    const int64_t count = ((m + 128 * t.cg - 1) / (128 * t.cg)) * ((n + t.bn - 1) / t.bn), units = sms / t.cg;
    // tiles that fill the GPU are not split (measured: the joining costs more than an even last wave gains)
    const int64_t most = may_split && count < units ? (blocks / 4 < 16 ? blocks / 4 : 16) : 1;
    for (int64_t s = 1; s == 1 || s <= most; ++s) {
      const int64_t per = (blocks + s - 1) / s;
      if (s > 1 && (blocks + per - 1) / per != s) continue;  // an empty part
      const int64_t waves = (count * s + units - 1) / units;
      const double load = (double)(count * s < units ? count * s : units) / units;
      const double per_block = t.alone + (t.busy - t.alone) * load;
      double us = waves * per * per_block + 2.0 * t.bn / 256;
      if (s > 1) us += 3.0 + (double)m * n * (4.0 * s * 2 + 2) * 1e-6 / 7.0;
      if (us < best_us) {
        best_us = us;
        best = {t.cg, t.bn, (int)s, (int)per};
      }
    }
  }
  return best;
}
static int64_t part_rows(const Plan &p, int64_t m) { return (m + 128 * p.cg - 1) / (128 * p.cg) * (128 * p.cg); }
static int64_t part_cols(const Plan &p, int64_t n) { return (n + p.bn - 1) / p.bn * p.bn; }
static size_t part_bytes(const Plan &p, int64_t m, int64_t n) {
  return p.splits > 1 ? (size_t)p.splits * part_rows(p, m) * part_cols(p, n) * sizeof(float) : 0;
}
static size_t round16(size_t n) { return (n + 15) / 16 * 16; }
// partial column sums of an [m][n] result: a row for every 32 of its rows
static size_t sums_bytes(int64_t m, int64_t n) { return round16((size_t)((m + 31) / 32) * n * sizeof(float)); }
// ... and of the activation-gradient pass: a row for every block of rows.  Two turns of 8 rows a block while
// that does not fill the GPU; few rows in one block, whose sums need no adding
static int row_blocks(int64_t rows, int64_t cols, int sms) {
  const int64_t across = (cols + 255) / 256, most = (8ll * sms + across - 1) / across, need = rows <= 64 ? 1 : (rows + 15) / 16;
  return (int)(need < most ? need : most);
}
template <typename T>
static int add_sums(const float *part, int parts, int cols, void *db, cudaStream_t st) {
  sums_kernel<T><<<(cols + 31) / 32, dim3(32, 32), 0, st>>>(part, parts, cols, static_cast<T *>(db));
  if (cudaGetLastError() != cudaSuccess) return KDA_ERR_CUDA;
  count_launch();
  return KDA_OK;
}
template <typename T, int ACT>
static int act_grad(int64_t rows, int64_t cols, const void *dy, int64_t ldy, const void *z, int64_t ldz, void *dz, int64_t ldd,
                    void *db, void *ws, int sms, cudaStream_t st) {
  const int blocks = row_blocks(rows, cols, sms);
  const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)blocks), block(32, 8);
  const T *y = static_cast<const T *>(dy), *zz = static_cast<const T *>(z);
  T *out = static_cast<T *>(dz);
  const int vy = tma_able(dy, ldy), vz = tma_able(z, ldz), vd = tma_able(dz, ldd);  // 16-byte rows
  float *part = static_cast<float *>(ws);
  if (db)
    act_grad_kernel<T, ACT, true><<<grid, block, 0, st>>>(rows, (int)cols, y, ldy, zz, ldz, out, ldd, vy, vz, vd, part,
                                                          static_cast<T *>(db));
  else
    act_grad_kernel<T, ACT, false><<<grid, block, 0, st>>>(rows, (int)cols, y, ldy, zz, ldz, out, ldd, vy, vz, vd, nullptr, nullptr);
  if (cudaGetLastError() != cudaSuccess) return KDA_ERR_CUDA;
  count_launch();
  return db && blocks > 1 ? add_sums<T>(part, blocks, (int)cols, db, st) : KDA_OK;
}
template <typename T>
static int act_grad(int act, int64_t rows, int64_t cols, const void *dy, int64_t ldy, const void *z, int64_t ldz, void *dz,
                    int64_t ldd, void *db, void *ws, int sms, cudaStream_t st) {
  switch (act) {
    case KDA_ACT_RELU: return act_grad<T, KDA_ACT_RELU>(rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
    case KDA_ACT_SILU: return act_grad<T, KDA_ACT_SILU>(rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
    case KDA_ACT_GELU: return act_grad<T, KDA_ACT_GELU>(rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
    case KDA_ACT_GELU_TANH: return act_grad<T, KDA_ACT_GELU_TANH>(rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
    default: return act_grad<T, KDA_ACT_NONE>(rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
  }
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN>
static int launch(Args &g, int sms, cudaStream_t st) {
  using S = Shape<CG, BN>;
  auto kernel = gemm_kernel<T, CG, BN, A_MN, B_MN>;
  g.tiles_m = (g.m + 128 * CG - 1) / (128 * CG);
  g.tiles_n = (g.n + BN - 1) / BN;
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  g.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
            ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
  static std::atomic<uint64_t> allowed{0};  // devices (of the first 64) where the kernel may use that much shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KDA_ERR_CUDA;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return KDA_ERR_CUDA;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t count = (int64_t)g.tiles_m * g.tiles_n * g.splits, units = sms / CG;
  if (count > (1ll << 30)) return KDA_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((count < units ? count : units) * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, g) != cudaSuccess) return KDA_ERR_CUDA;
  count_launch();
  return KDA_OK;
}

// One product: the tiles (and parts), then whatever of parts and column sums is left to add.  The
// workspace holds the column sums' partials, then the parts.
template <typename T, bool A_MN, bool B_MN>
static int run(Args &g, const Plan &p, const void *a, int64_t lda, const void *b, int64_t ldb, void *ws, void *db, int sms,
               cudaStream_t st) {
  int s;
  if ((s = A_MN ? tma_map_rows16(&g.a, a, g.k, g.m, lda, 64) : tma_map_rows16(&g.a, a, g.m, g.k, lda, 128))) return s;
  if ((s = B_MN ? tma_map_rows16(&g.b, b, g.k, g.n, ldb, 64) : tma_map_rows16(&g.b, b, g.n, g.k, ldb, p.bn / p.cg))) return s;
  g.splits = p.splits;
  g.per_split = p.per_split;
  char *at = static_cast<char *>(ws);
  if (db) {
    g.sums = reinterpret_cast<float *>(at);
    at += sums_bytes(g.m, g.n);
  }
  const int64_t rows = part_rows(p, g.m);
  if (p.splits > 1) {
    g.part = reinterpret_cast<float *>(at);
    g.ldp = part_cols(p, g.n);
    if ((s = tma_map_rows32(&g.out, at, p.splits * rows, g.ldp, g.ldp, 32))) return s;
  }
  s = p.cg == 2    ? launch<T, 2, 256, A_MN, B_MN>(g, sms, st)
      : p.bn == 128 ? launch<T, 1, 128, A_MN, B_MN>(g, sms, st)
                    : launch<T, 1, 64, A_MN, B_MN>(g, sms, st);
  if (s) return s;
  if (p.splits > 1) {
    const int col_blocks = (g.n + 511) / 512;
    const int per = db ? 32 : kJoinRows;
    const unsigned blocks = (unsigned)((int64_t)((g.m + per - 1) / per) * col_blocks);
    if (db) join_kernel<T, true><<<blocks, dim3(64, 4), 0, st>>>(g, rows, col_blocks);
    else join_kernel<T, false><<<blocks, dim3(64, 4), 0, st>>>(g, rows, col_blocks);
    if (cudaGetLastError() != cudaSuccess) return KDA_ERR_CUDA;
    count_launch();
  }
  return db ? add_sums<T>(g.sums, (g.m + 31) / 32, g.n, db, st) : KDA_OK;
}

template <typename T, int MT, int NB>
static int few_rows(const FewArgs &a, int sms, cudaStream_t st) {
  // warps per group of outputs: the fewest within a tenth of the least time, waves of CTAs by a warp's share of k
  // (16 x 11008 x 4096: two warps 25.0 us, four, whose CTAs leave a second wave of 48, 28.0)
  const int groups = (a.n + 8 * NB - 1) / (8 * NB);
  int kw = 1;
  auto time = [&](int w) { return (double)(((int64_t)groups * w + 2 * kFewWarps * sms - 1) / (2 * kFewWarps * sms)) / w; };
  for (int w = 2; w <= kFewWarps; w *= 2)
    if (time(w) < 0.9 * time(kw)) kw = w;
  const int range = ((a.k + 31) / 32 + kw - 1) / kw * 32, per = kFewWarps / kw;
  few_rows_kernel<T, MT, NB><<<(groups + per - 1) / per, 32 * kFewWarps, 0, st>>>(a, kw, range);
  if (cudaGetLastError() != cudaSuccess) return KDA_ERR_CUDA;
  count_launch();
  return KDA_OK;
}
template <typename T>
static int few_rows(const FewArgs &a, int sms, cudaStream_t st) {
  // eight outputs a warp where their CTAs, eight warps for each, are resident at once (with more than 16 rows: one an
  // SM), sixteen where they are not: 16 x 512 x 2048 3.6 us by eight, 4.6 by sixteen, 16 x 2048 x 8192 10.9
  // and 12.0, 16 x 8192 x 2048 11.2 and 9.8, 1 x 8192 x 2048 8.9 and 7.9, 32 x 1024 x 4096 7.2 and 8.5
  const bool narrow = (a.n + 7) / 8 <= (a.m <= 16 ? 2 : 1) * sms;
  if (narrow) return a.m <= 8 ? few_rows<T, 1, 1>(a, sms, st) : a.m <= 16 ? few_rows<T, 2, 1>(a, sms, st) : few_rows<T, 4, 1>(a, sms, st);
  return a.m <= 8 ? few_rows<T, 1, 2>(a, sms, st) : a.m <= 16 ? few_rows<T, 2, 2>(a, sms, st) : few_rows<T, 4, 2>(a, sms, st);
}

static int set_out(Args &g, void *p, int64_t ld) {
  g.out_ptr = p;
  g.ldo = ld;
  g.out_tma = tma_able(p, ld);
  return g.out_tma ? tma_map_rows16(&g.out, p, g.m, g.n, ld, 32) : KDA_OK;
}
static int set_in(Args &g, int kind, const void *p, int64_t ld) {
  g.in_kind = kind;
  g.in_ptr = p;
  g.ldi = ld;
  g.in_tma = tma_able(p, ld);
  return g.in_tma ? tma_map_rows16(&g.in, p, g.m, g.n, ld, 32) : KDA_OK;
}

static int check(int dtype, int act, int64_t m, int64_t n, int64_t k) {
  if (dtype != KDA_BF16 && dtype != KDA_F16) return KDA_ERR_DTYPE;
  if (act < KDA_ACT_NONE || act > KDA_ACT_GELU_TANH) return KDA_ERR_INVALID_ARG;
  if (m <= 0 || n <= 0 || k <= 0) return KDA_ERR_INVALID_ARG;
  if (m > (1ll << 30) || n > (1ll << 30) || k > (1ll << 30)) return KDA_ERR_UNSUPPORTED;
  return KDA_OK;
}
static bool ld_ok(int64_t ld, int64_t cols) { return ld >= cols && ld <= (1ll << 38); }
static bool even(std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if ((uintptr_t)p % 2) return false;
  return true;
}

// The plan for a product, and whether the workspace holds it; without one k is not split.
static int plan_in(Plan &p, int64_t m, int64_t n, int64_t k, int sms, bool sums, const void *ws, size_t ws_bytes) {
  p = plan_for(m, n, k, sms, ws != nullptr);
  const size_t need = part_bytes(p, m, n) + (sums ? sums_bytes(m, n) : 0);
  return need && (!ws || (uintptr_t)ws % 16 || ws_bytes < need) ? KDA_ERR_WORKSPACE : KDA_OK;
}

int device_status(bool reset) {
  int v = 0;
  const int zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return KDA_ERR_CUDA;
  if (cudaMemcpyFromSymbol(&v, g_linear_status, sizeof(v)) != cudaSuccess) return KDA_ERR_CUDA;
  if (reset && v && cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(zero)) != cudaSuccess) return KDA_ERR_CUDA;
  return v;
}

}  // namespace linear
int linear_device_status(bool reset) { return linear::device_status(reset); }
}  // namespace kda

using namespace kda::linear;

extern "C" {

size_t kda_linear_workspace_bytes(int op, int64_t M, int64_t N, int64_t K, int with_db) {
  if (check(KDA_BF16, KDA_ACT_NONE, M, N, K)) return 0;
  int sms = device_sms();
  if (!sms) sms = 148;  // no device: the size on a B200
  if (op == KDA_LINEAR_FWD) return is_few(M, N, sms) ? 0 : part_bytes(plan_for(M, N, K, sms, true), M, N);
  if (op == KDA_LINEAR_DGRAD) return part_bytes(plan_for(M, K, N, sms, true), M, K) + (with_db ? sums_bytes(M, K) : 0);
  if (op == KDA_LINEAR_WGRAD) return part_bytes(plan_for(N, K, M, sms, true), N, K);
  if (op == KDA_LINEAR_ACT_GRAD) return with_db ? round16((size_t)row_blocks(M, N, sms) * N * sizeof(float)) : 0;
  return 0;
}

int kda_linear_fwd(int dtype, int act, int64_t M, int64_t N, int64_t K, const void *x, int64_t ldx, const void *w,
                   int64_t ldw, const void *bias, const void *residual, int64_t ldr, void *y, int64_t ldy, void *z,
                   int64_t ldz, void *ws, size_t ws_bytes, void *stream) {
  int s = check(dtype, act, M, N, K);
  if (s) return s;
  if (!x || !w || !y || !ld_ok(ldx, K) || !ld_ok(ldw, K) || !ld_ok(ldy, N) || (residual && !ld_ok(ldr, N)) ||
      (z && !ld_ok(ldz, N)))
    return KDA_ERR_INVALID_ARG;
  if (!tma_able(x, ldx) || !tma_able(w, ldw) || (z && !tma_able(z, ldz)) || !even({bias, residual, y}))
    return KDA_ERR_MISALIGNED;
  const int sms = device_sms();
  if (!sms) return KDA_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  if (is_few(M, N, sms)) {
    const FewArgs a = {x, w, bias, residual, y, z, ldx, ldw, ldr, ldy, ldz, (int)M, (int)N, (int)K, act};
    return dtype == KDA_BF16 ? few_rows<__nv_bfloat16>(a, sms, st) : few_rows<__half>(a, sms, st);
  }
  Plan p;
  if ((s = plan_in(p, M, N, K, sms, 0, ws, ws_bytes))) return s;
  Args g = {};
  g.m = (int)M; g.n = (int)N; g.k = (int)K; g.act = act; g.bias = bias;
  if ((s = set_out(g, y, ldy))) return s;
  if (residual && (s = set_in(g, kInAdd, residual, ldr))) return s;
  if (z) {
    g.save_z = 1;
    g.z_ptr = z;
    g.ldz = ldz;
    if ((s = kda::tma_map_rows16(&g.z, z, M, N, ldz, 32))) return s;
  }
  return dtype == KDA_BF16 ? run<__nv_bfloat16, false, false>(g, p, x, ldx, w, ldw, ws, nullptr, sms, st)
                           : run<__half, false, false>(g, p, x, ldx, w, ldw, ws, nullptr, sms, st);
}

int kda_linear_dgrad(int dtype, int act, int64_t M, int64_t N, int64_t K, const void *dz, int64_t ldd, const void *w,
                     int64_t ldw, const void *z, int64_t ldz, void *dx, int64_t ldx, void *db, void *ws,
                     size_t ws_bytes, void *stream) {
  int s = check(dtype, act, M, N, K);
  if (s) return s;
  if (!dz || !w || !dx || !ld_ok(ldd, N) || !ld_ok(ldw, K) || !ld_ok(ldx, K) || (z && !ld_ok(ldz, K)) ||
      (act != KDA_ACT_NONE && !z))
    return KDA_ERR_INVALID_ARG;
  if (!tma_able(dz, ldd) || !tma_able(w, ldw) || !even({z, dx, db})) return KDA_ERR_MISALIGNED;
  if (db && !ws) return KDA_ERR_WORKSPACE;
  const int sms = device_sms();
  if (!sms) return KDA_ERR_CUDA;
  Plan p;
  if ((s = plan_in(p, M, K, N, sms, db != nullptr, ws, ws_bytes))) return s;
  Args g = {};
  g.m = (int)M; g.n = (int)K; g.k = (int)N; g.act = act;
  if ((s = set_out(g, dx, ldx))) return s;
  if (act != KDA_ACT_NONE && (s = set_in(g, kInActGrad, z, ldz))) return s;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == KDA_BF16 ? run<__nv_bfloat16, false, true>(g, p, dz, ldd, w, ldw, ws, db, sms, st)
                           : run<__half, false, true>(g, p, dz, ldd, w, ldw, ws, db, sms, st);
}

int kda_linear_wgrad(int dtype, int64_t M, int64_t N, int64_t K, const void *dz, int64_t ldd, const void *x, int64_t ldx,
                     void *dw, int64_t ldw, void *ws, size_t ws_bytes, void *stream) {
  int s = check(dtype, KDA_ACT_NONE, M, N, K);
  if (s) return s;
  if (!dz || !x || !dw || !ld_ok(ldd, N) || !ld_ok(ldx, K) || !ld_ok(ldw, K)) return KDA_ERR_INVALID_ARG;
  if (!tma_able(dz, ldd) || !tma_able(x, ldx) || !even({dw})) return KDA_ERR_MISALIGNED;
  const int sms = device_sms();
  if (!sms) return KDA_ERR_CUDA;
  Plan p;
  if ((s = plan_in(p, N, K, M, sms, false, ws, ws_bytes))) return s;
  Args g = {};
  g.m = (int)N; g.n = (int)K; g.k = (int)M;
  if ((s = set_out(g, dw, ldw))) return s;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == KDA_BF16 ? run<__nv_bfloat16, true, true>(g, p, dz, ldd, x, ldx, ws, nullptr, sms, st)
                           : run<__half, true, true>(g, p, dz, ldd, x, ldx, ws, nullptr, sms, st);
}

int kda_act_grad(int dtype, int act, int64_t rows, int64_t cols, const void *dy, int64_t ldy, const void *z, int64_t ldz,
                 void *dz, int64_t ldd, void *db, void *ws, size_t ws_bytes, void *stream) {
  int s = check(dtype, act, rows, cols, 1);
  if (s) return s;
  if (!dy || (!dz && !db) || !ld_ok(ldy, cols) || (dz && !ld_ok(ldd, cols)) || (z && !ld_ok(ldz, cols)) ||
      (act != KDA_ACT_NONE && !z))
    return KDA_ERR_INVALID_ARG;
  if (!even({dy, z, dz, db})) return KDA_ERR_MISALIGNED;
  if (db && (!ws || (uintptr_t)ws % 16)) return KDA_ERR_WORKSPACE;
  const int sms = device_sms();
  if (!sms) return KDA_ERR_CUDA;
  if (db && ws_bytes < round16((size_t)row_blocks(rows, cols, sms) * cols * sizeof(float))) return KDA_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == KDA_BF16 ? act_grad<__nv_bfloat16>(act, rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st)
                           : act_grad<__half>(act, rows, cols, dy, ldy, z, ldz, dz, ldd, db, ws, sms, st);
}

}  // extern "C"
