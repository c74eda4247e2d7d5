// The matrix product behind the gated feed-forward block: D = A B^T in 16-bit types with fp32 sums on tcgen05, operands by bulk
// tensor copies, the element-wise work around the product in its epilogue.  gated_mlp.cu has the operators and the reasons for
// the tiles.
//
// Two CTAs of a cluster work on one 256 x kN tile (cta_group::2): each holds 128 rows of A and half of B's rows in its shared memory
// and 128 rows of the result in its tensor memory, so that a byte from L2 serves twice the products that a CTA alone would
// get from it.  Warp 0 copies, warp 1 of the even CTA issues the products, warps 4-11 of both store the result: they work on one
// of two accumulators while the products of the next tile fill the other.  The CTAs walk the tiles with the stride of the grid.
//
// An operand is stored with its contracted dimension innermost ("K-major": A (M, K), B (N, K)) or outermost (MN-major: A (K, M),
// B (K, N)); both land as boxes of 64 lines of 128 bytes that the shared-memory descriptors describe.  Boxes beyond the matrix are
// zeros: no size but the multiple of 8 elements of a row matters.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "sm100_primitives.cuh"
#include "tensor_map.cuh"

namespace mf {
namespace gemm {

__device__ int32_t g_gemm_status = 0;  // MF_ERR_DEVICE_TIMEOUT after an expired wait

enum Epilogue { kGate, kGateGrad, kStore, kStoreF32 };

constexpr int kBlockK = 64;                       // elements of the contracted dimension in a stage
constexpr int kBoxBytes = 64 * 128;               // 64 lines of 64 16-bit elements
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (4 + kEpilogueWarps);
constexpr int kStageBuffer = 32 * 128;            // what a warp hands to the copy engine at once: 32 rows of 128 bytes
constexpr int kMaxSmem = 232448;

template <int kN, Epilogue kEpi>
struct Shape {
  static constexpr int kBoxesA = 2, kBoxesB = kN / 2 / 64;  // of one CTA
  static constexpr int kStageBytes = (kBoxesA + kBoxesB) * kBoxBytes;
  static constexpr int kBuffers = kEpi == kGateGrad ? 4 : kEpi == kGate ? 3 : 2;  // of 4 KB for each storing warp
  static constexpr int kBufferBytes = kEpilogueWarps * kBuffers * kStageBuffer;
  static constexpr int kStages = (kMaxSmem - 1024 - 1024 - kBufferBytes) / kStageBytes < 8 ? (kMaxSmem - 1024 - 1024 - kBufferBytes) / kStageBytes : 8;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kBufferBytes;
  static_assert(kStages >= 3, "too few stages");
  static constexpr int kTmemCols = 2 * kN;
};

struct Params {
  CUtensorMap a, b;         // boxes of 64 lines; b: of the even CTA's half where the halves are different matrices (kGate)
  CUtensorMap b2;           // kGate: the odd CTA's (the rows of the up projection)
  CUtensorMap out, out2;    // boxes of 32 lines.  kGate: hidden | -;  kGateGrad: gradients of gate | up;  else the result
  CUtensorMap pre, pre2;    // pre-activations of gate | up (kGate: written if keep_pre; kGateGrad: read)
  const void* bias;         // kGate: (2 F), kStore: (N); may be null
  float* column_sums;       // kGateGrad: (ceil(M / 32), 2 F) partial sums of the stored rows, or null
  int m, n, k;              // kGate, kGateGrad: n = F
  int splits, k_blocks_per_split;  // kStoreF32: the contracted dimension in `splits` pieces, each with a plane of its own
  int activation;
  int keep_pre;
  BoundedWaits waits;       // kinds: 0 operands, 1 stages, 2 accumulators, 3 drained accumulators
};

// ---- two-CTA forms -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_alloc2(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish2() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void umma2(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// Arrives on the barrier at this address in both CTAs once the products issued so far are done.
__device__ __forceinline__ void umma_commit2(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}
// One 64 x 64 box into this CTA; its bytes are counted on the barrier `bar` (a cluster address) of the even CTA.
__device__ __forceinline__ void load_box2(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void load_box(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_dst),
               "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t smem_src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_src)
               : "memory");
}
__device__ __forceinline__ void store_box3(const CUtensorMap* map, uint32_t smem_src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z),
               "r"(smem_src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// ---- element types -------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }

// kind::f16 with fp32 sums: D format (bits 4-5) 1 = f32, A (7-9) and B (10-12) 0 = f16, 1 = bf16
template <typename T, bool kAMn, bool kBMn, int kN>
__host__ __device__ constexpr uint32_t instruction() {
  constexpr uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)kAMn << 15) | ((uint32_t)kBMn << 16) | ((uint32_t)(kN >> 3) << 17) | ((256u >> 4) << 24);
}

// ---- activations ---------------------------------------------------------------------------------------------------
// act(z) = z s(w(z)) with the logistic function s: w = z is SiLU; w = 2 sqrt(2/pi) (z + 0.044715 z^3) is GELU in its tanh form, since
// (1 + tanh(a)) / 2 = s(2 a), and nothing cancels for large negative z.  The derivative is s + z s (1 - s) w'.
// Beyond |z| = 64 both are 0 or z (1 for the derivative) in fp32: the clamp keeps the cube and w' finite.
struct Act {
  float value, slope;
};
template <bool kSlope>
__device__ __forceinline__ Act activation(float z, int kind) {
  float w = z, dw = 1.f;
  if (kind == MF_ACT_GELU_TANH) {
    const float c = fminf(fmaxf(z, -64.f), 64.f), c2 = c * c;
    w = 1.5957691216057308f * c * (1.f + 0.044715f * c2);
    dw = 1.5957691216057308f * (1.f + 3.f * 0.044715f * c2);
  }
  const float s = __fdividef(1.f, 1.f + __expf(-w));
  Act r;
  r.value = z * s;
  r.slope = kSlope ? s + r.value * (1.f - s) * dw : 0.f;
  return r;
}

// Eight values of a bias from column c on (a multiple of 8); zeros behind the last.
template <typename T>
__device__ __forceinline__ void bias8(const T* bias, int c, int n, float (&b)[8]) {
  const uint4 v = c < n ? __ldg(reinterpret_cast<const uint4*>(bias + c)) : make_uint4(0u, 0u, 0u, 0u);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(w[i]);
    b[2 * i] = f.x, b[2 * i + 1] = f.y;
  }
}

// Where 16 bytes `chunk` of line `row` of a box lie.
__device__ __forceinline__ uint32_t box_chunk(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

// Tiles are walked in groups of rows that stay in L2 together: all columns of kGroup row tiles, the row tiles fastest.
constexpr int kGroup = 8;
struct Tile {
  int m, n, split;
};
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n) {
  Tile r;
  const int plane = tiles_m * tiles_n;
  r.split = t / plane;
  t -= r.split * plane;
  const int group = t / (kGroup * tiles_n), first = group * kGroup, rows = min(kGroup, tiles_m - first);
  t -= first * tiles_n;
  r.m = first + t % rows;
  r.n = t / rows;
  return r;
}

template <typename T, bool kAMn, bool kBMn, int kN, Epilogue kEpi>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Params p) {
  using Sh = Shape<kN, kEpi>;
  constexpr int kStages = Sh::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ uint64_t bar_full[kStages], bar_empty[kStages], bar_acc[2], bar_drained[2], bar_in[2 * kEpilogueWarps], bar_end;
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  constexpr int kTileN = kEpi == kGate ? kN / 2 : kN;  // columns of the result in a tile
  const int tiles_m = (p.m + 255) / 256, tiles_n = (p.n + kTileN - 1) / kTileN;
  const int tiles = tiles_m * tiles_n * p.splits;
  const int k_blocks = (p.k + kBlockK - 1) / kBlockK;

  if (threadIdx.x == 0) {
    const int w = p.waits.withheld;
    for (int i = 0; i < kStages; ++i) mbar_init(&bar_full[i], 1 + (w == 0)), mbar_init(&bar_empty[i], 1 + (w == 1));
    for (int i = 0; i < 2; ++i) mbar_init(&bar_acc[i], 1 + (w == 2)), mbar_init(&bar_drained[i], 2 * kEpilogueWarps + (w == 3));
    for (int i = 0; i < 2 * kEpilogueWarps; ++i) mbar_init(&bar_in[i], 1);
    mbar_init(&bar_end, 1);
    mbar_fence_init();
  }
  if (warp == 2) {
    tmem_alloc2(&tmem_base_s, Sh::kTmemCols);
    tmem_relinquish2();
  }
  tc_fence_before_sync();
  cluster_sync();  // the barriers of both CTAs are ready
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;
  launch_dependents();
  wait_for_previous();

  bool bad = false;
  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (elect_one()) {
      uint32_t it = 0;
      for (int t = pair; t < tiles && !bad; t += pairs) {
        const Tile tile = tile_at(t, tiles_m, tiles_n);
        const int kb0 = tile.split * p.k_blocks_per_split, kb1 = min(k_blocks, kb0 + p.k_blocks_per_split);
        const int row = tile.m * 256 + 128 * (int)rank;
        const CUtensorMap* bmap = kEpi == kGate && rank ? &p.b2 : &p.b;
        const int col = kEpi == kGate ? tile.n * kTileN : tile.n * kN + (kN / 2) * (int)rank;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % kStages;
          const uint32_t phase = (it / kStages) & 1;
          if (it >= kStages && !mbar_wait_for(&bar_empty[s], phase ^ 1, p.waits.limit)) {
            bad = true;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&bar_full[s], 2 * Sh::kStageBytes);
          const uint32_t bar = map_to_rank(smem_u32(&bar_full[s]), 0), dst = smem + s * Sh::kStageBytes;
#pragma unroll
          for (int i = 0; i < Sh::kBoxesA; ++i)
            load_box2(dst + i * kBoxBytes, &p.a, kAMn ? row + 64 * i : kb * kBlockK, kAMn ? kb * kBlockK : row + 64 * i, bar);
#pragma unroll
          for (int i = 0; i < Sh::kBoxesB; ++i)
            load_box2(dst + (Sh::kBoxesA + i) * kBoxBytes, bmap, kBMn ? col + 64 * i : kb * kBlockK, kBMn ? kb * kBlockK : col + 64 * i, bar);
        }
      }
      if (bad && rank == 0) {  // copies that still fly write to these CTAs: their bytes arrive here (once a wait has lasted its second, all have)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
          if (!mbar_wait(&bar_full[i % kStages], (i / kStages) & 1)) break;
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---------------------------------------------------------------- products
    if (elect_one()) {
      constexpr uint32_t idesc = instruction<T, kAMn, kBMn, kN>();
      // K-major: 16 elements of a line further on; MN-major: 16 lines further on, 64-wide chunks a box apart
      constexpr uint32_t kStepA = kAMn ? 16 * 128 : 32, kStepB = kBMn ? 16 * 128 : 32;
      const uint64_t a0 = make_smem_desc_sw128(smem, kAMn ? kBoxBytes : 0, 1024);
      const uint64_t b0 = make_smem_desc_sw128(smem + Sh::kBoxesA * kBoxBytes, kBMn ? kBoxBytes : 0, 1024);
      uint32_t it = 0;
      int n = 0;
      for (int t = pair; t < tiles && !bad; t += pairs, ++n) {
        const Tile tile = tile_at(t, tiles_m, tiles_n);
        const int kb0 = tile.split * p.k_blocks_per_split, kb1 = min(k_blocks, kb0 + p.k_blocks_per_split);
        const int buf = n & 1;
        if (n >= 2 && !mbar_wait_for(&bar_drained[buf], ((n >> 1) & 1) ^ 1, p.waits.limit)) {
          bad = true;
          break;
        }
        tc_fence_after_sync();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait_for(&bar_full[s], (it / kStages) & 1, p.waits.limit)) {
            bad = true;
            break;
          }
          tc_fence_after_sync();
          const uint64_t a = desc_advance(a0, s * Sh::kStageBytes), b = desc_advance(b0, s * Sh::kStageBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / 16; ++k)
            umma2(tmem + buf * kN, desc_advance(a, k * kStepA), desc_advance(b, k * kStepB), idesc, kb > kb0 || k > 0);
          umma_commit2(&bar_empty[s]);
        }
        if (!bad) umma_commit2(&bar_acc[buf]);
      }
      if (bad) {  // no product may still run when the tensor memory is freed
        umma_commit2(&bar_end);
        mbar_wait(&bar_end, 0);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- results
    const int ew = warp - 4, quad = warp & 3, half = ew >> 2;
    const uint32_t buffers = smem + kStages * Sh::kStageBytes + ew * Sh::kBuffers * kStageBuffer;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quad) << 16);
    int n = 0;
    uint32_t chunk = 0, fetched = 0;  // chunks of columns, counted over all tiles
    constexpr int kHalf = kTileN / 2;              // columns of the result that this warp stores
    constexpr int kChunks = kHalf / 64;

    // the pre-activations of chunk c of tile t, the i-th in all, on their way to buffers 2 (i & 1) and 2 (i & 1) + 1
    auto fetch = [&](int t, int c) {
      const uint32_t i = fetched++;
      const Tile tile = tile_at(t, tiles_m, tiles_n);
      const int row = tile.m * 256 + 128 * (int)rank + 32 * quad, col = tile.n * kTileN + half * kHalf + 64 * c;
      uint64_t* bar = &bar_in[2 * ew + (i & 1)];
      const uint32_t dst = buffers + 2 * (i & 1) * kStageBuffer;
      mbar_arrive_expect_tx(bar, 2 * kStageBuffer);
      load_box(dst, &p.pre, col, row, bar);
      load_box(dst + kStageBuffer, &p.pre2, col, row, bar);
    };
    if (kEpi == kGateGrad && pair < tiles && lane == 0) fetch(pair, 0);

    for (int t = pair; t < tiles; t += pairs, ++n) {
      const Tile tile = tile_at(t, tiles_m, tiles_n);
      const int row0 = tile.m * 256 + 128 * (int)rank + 32 * quad, col0 = tile.n * kTileN + half * kHalf;
      const int buf = n & 1;
      if (!mbar_wait_for(&bar_acc[buf], (n >> 1) & 1, p.waits.limit)) bad = true;
      bad = __any_sync(0xffffffffu, bad);
      if (bad) break;
      tc_fence_after_sync();
      const uint32_t acc = lane_base + buf * kN;

      if constexpr (kEpi == kGate) {
        const T* bias = static_cast<const T*>(p.bias);
        if (lane == 0) store_wait_read<0>();  // of the tile before
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t g[32], u[32];
          tmem_ld32(acc + half * kHalf + 32 * c, g);
          tmem_ld32(acc + kTileN + half * kHalf + 32 * c, u);
          tmem_ld_wait();
          if (c == 1) {
            tc_fence_before_sync();
            if (lane == 0) arrive_cluster(map_to_rank(smem_u32(&bar_drained[buf]), 0));
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float bg[8] = {}, bu[8] = {};
            if (bias) {
              bias8(bias, col0 + 32 * c + 8 * v, p.n, bg);
              bias8(bias + p.n, col0 + 32 * c + 8 * v, p.n, bu);
            }
            uint32_t hw[4], gw[4], uw[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float g0 = __uint_as_float(g[8 * v + 2 * e]) + bg[2 * e], g1 = __uint_as_float(g[8 * v + 2 * e + 1]) + bg[2 * e + 1];
              const float u0 = __uint_as_float(u[8 * v + 2 * e]) + bu[2 * e], u1 = __uint_as_float(u[8 * v + 2 * e + 1]) + bu[2 * e + 1];
              hw[e] = pack2<T>(activation<false>(g0, p.activation).value * u0, activation<false>(g1, p.activation).value * u1);
              gw[e] = pack2<T>(g0, g1), uw[e] = pack2<T>(u0, u1);
            }
            const uint32_t at = buffers + box_chunk(lane, 4 * c + v);
            sts128(at, make_uint4(hw[0], hw[1], hw[2], hw[3]));
            if (p.keep_pre) {
              sts128(at + kStageBuffer, make_uint4(gw[0], gw[1], gw[2], gw[3]));
              sts128(at + 2 * kStageBuffer, make_uint4(uw[0], uw[1], uw[2], uw[3]));
            }
          }
        }
        fence_smem_to_async_proxy();
        __syncwarp();
        if (lane == 0 && row0 < p.m && col0 < p.n) {
          store_box(&p.out, buffers, col0, row0);
          if (p.keep_pre) {
            store_box(&p.pre, buffers + kStageBuffer, col0, row0);
            store_box(&p.pre2, buffers + 2 * kStageBuffer, col0, row0);
          }
          store_commit();
        }
      } else if constexpr (kEpi == kGateGrad) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c, ++chunk) {
          // the next chunk's pre-activations, once the buffers' previous results have left
          const bool last = c == kChunks - 1;
          if (lane == 0 && (!last || t + pairs < tiles)) {
            store_wait_read<0>();
            fetch(last ? t + pairs : t, last ? 0 : c + 1);
          }
          if (!mbar_wait_for(&bar_in[2 * ew + (chunk & 1)], (chunk >> 1) & 1, p.waits.limit)) bad = true;
          bad = __any_sync(0xffffffffu, bad);
          if (bad) break;
          const uint32_t gate = buffers + 2 * (chunk & 1) * kStageBuffer, up = gate + kStageBuffer;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t d[32];
            tmem_ld32(acc + half * kHalf + 64 * c + 32 * h, d);
            tmem_ld_wait();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const uint32_t at = box_chunk(lane, 4 * h + v);
              const uint4 gw = lds128(gate + at), uw = lds128(up + at);
              const uint32_t gs[4] = {gw.x, gw.y, gw.z, gw.w}, us[4] = {uw.x, uw.y, uw.z, uw.w};
              uint32_t dg[4], du[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 g = unpack2<T>(gs[e]), u = unpack2<T>(us[e]);
                const float d0 = __uint_as_float(d[8 * v + 2 * e]), d1 = __uint_as_float(d[8 * v + 2 * e + 1]);
                const Act a0 = activation<true>(g.x, p.activation), a1 = activation<true>(g.y, p.activation);
                dg[e] = pack2<T>(d0 * u.x * a0.slope, d1 * u.y * a1.slope);
                du[e] = pack2<T>(d0 * a0.value, d1 * a1.value);
              }
              sts128(gate + at, make_uint4(dg[0], dg[1], dg[2], dg[3]));
              sts128(up + at, make_uint4(du[0], du[1], du[2], du[3]));
            }
          }
          if (last) {
            tc_fence_before_sync();
            if (lane == 0) arrive_cluster(map_to_rank(smem_u32(&bar_drained[buf]), 0));
          }
          fence_smem_to_async_proxy();
          __syncwarp();
          const int col = col0 + 64 * c;
          if (lane == 0 && row0 < p.m && col < p.n) {
            store_box(&p.out, gate, col, row0);
            store_box(&p.out2, up, col, row0);
            store_commit();
          }
          if (p.column_sums && row0 < p.m) {  // of the values as stored: a lane adds two columns of the 32 rows (rows beyond the last are zeros)
#pragma unroll
            for (int side = 0; side < 2; ++side) {
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int r = 0; r < 32; ++r) {
                const float2 v = unpack2<T>(lds32((side ? up : gate) + box_chunk(r, lane >> 2) + 4 * (lane & 3)));
                sum.x += v.x, sum.y += v.y;
              }
              const int cc = col + 2 * lane;
              if (cc < p.n) *reinterpret_cast<float2*>(p.column_sums + (size_t)(row0 >> 5) * (2 * (size_t)p.n) + side * (size_t)p.n + cc) = sum;
            }
            __syncwarp();
          }
        }
        if (bad) break;
      } else if constexpr (kEpi == kStore) {
        const T* bias = static_cast<const T*>(p.bias);
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c, ++chunk) {
          uint32_t words[32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t d[32];
            tmem_ld32(acc + half * kHalf + 64 * c + 32 * h, d);
            tmem_ld_wait();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float b[8] = {};
              if (bias) bias8(bias, col0 + 64 * c + 32 * h + 8 * v, p.n, b);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                words[16 * h + 4 * v + e] = pack2<T>(__uint_as_float(d[8 * v + 2 * e]) + b[2 * e], __uint_as_float(d[8 * v + 2 * e + 1]) + b[2 * e + 1]);
            }
          }
          if (c == kChunks - 1) {
            tc_fence_before_sync();
            if (lane == 0) arrive_cluster(map_to_rank(smem_u32(&bar_drained[buf]), 0));
          }
          const uint32_t dst = buffers + (chunk & 1) * kStageBuffer;
          if (lane == 0) store_wait_read<1>();
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 8; ++v) sts128(dst + box_chunk(lane, v), make_uint4(words[4 * v], words[4 * v + 1], words[4 * v + 2], words[4 * v + 3]));
          fence_smem_to_async_proxy();
          __syncwarp();
          if (lane == 0 && row0 < p.m && col0 + 64 * c < p.n) {
            store_box(&p.out, dst, col0 + 64 * c, row0);
            store_commit();
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < kHalf / 32; ++c, ++chunk) {
          uint32_t d[32];
          tmem_ld32(acc + half * kHalf + 32 * c, d);
          tmem_ld_wait();
          if (c == kHalf / 32 - 1) {
            tc_fence_before_sync();
            if (lane == 0) arrive_cluster(map_to_rank(smem_u32(&bar_drained[buf]), 0));
          }
          const uint32_t dst = buffers + (chunk & 1) * kStageBuffer;
          if (lane == 0) store_wait_read<1>();
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 8; ++v) sts128(dst + box_chunk(lane, v), make_uint4(d[4 * v], d[4 * v + 1], d[4 * v + 2], d[4 * v + 3]));
          fence_smem_to_async_proxy();
          __syncwarp();
          if (lane == 0 && row0 < p.m && col0 + 32 * c < p.n) {
            store_box3(&p.out, dst, col0 + 32 * c, row0, tile.split);
            store_commit();
          }
        }
      }
    }
    if (lane == 0) {
      if (kEpi == kGateGrad && bad)  // pre-activations that still fly
        for (uint32_t i = fetched > 2 ? fetched - 2 : 0; i < fetched; ++i)
          if (!mbar_wait(&bar_in[2 * ew + (i & 1)], (i >> 1) & 1)) break;
      store_wait_all();
    }
  }
  if (bad) atomicExch(&g_gemm_status, MF_ERR_DEVICE_TIMEOUT);
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();  // no arrival, copy or product of either CTA is outstanding
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc2(tmem, Sh::kTmemCols);
  }
}

}  // namespace gemm
}  // namespace mf
