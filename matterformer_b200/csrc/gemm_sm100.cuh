// The matrix product behind the gated feed-forward block: D = A B^T in 16-bit types with fp32 sums on tcgen05, operands by bulk
// tensor copies, the element-wise work around the product in its epilogue.  gated_mlp.cu has the operators and the reasons for
// the tiles.
//
// Two CTAs of a cluster work on one 256 x 256 tile (cta_group::2): each holds 128 rows of A and half of B's rows in its shared memory
// and 128 rows of the result in its tensor memory, so that a byte from L2 serves twice the products that a CTA alone would
// get from it.  Warp 0 copies, warp 1 of the even CTA issues the products, warps 4-11 of both store the result: they work on one
// of two accumulators while the products of the next tile fill the other.  The CTAs walk the tiles with the stride of the grid.
// 256 columns at 8192 x 2048 x 4096: 95 us, 1441 TFLOP/s (cuBLAS at 8192^3: 1644); 128 columns: 108 us, the copies bound it.
//
// A last round of tiles that would leave half of the pairs or more without work is cut into tiles of 128 or 64 columns.
//
// An operand is stored with its contracted dimension innermost ("K-major": A (M, K), B (N, K)) or outermost (MN-major: A (K, M),
// B (K, N)); both land as boxes of 64 lines of 128 bytes that the shared-memory descriptors describe.  Boxes beyond the matrix are
// zeros: no size but the multiple of 8 elements of a row matters.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "gated_mlp.cuh"
#include "sm100_primitives.cuh"
#include "tensor_map.cuh"

namespace mf {
namespace gemm {

// MF_ERR_DEVICE_TIMEOUT after an expired wait, until it is read: of calls | of the self-test
__device__ int32_t g_gemm_status[2] = {0, 0};

// kGate: two projections, activation and product; kGateKeep: the pre-activations are stored as well; kGateGrad: the gradient of both;
// kStore: the product and a bias; kGradients: the weights' gradients, two products over the same long dimension (of operands that have it
// outermost), and the input's, side by side
enum Epilogue { kGate, kGateKeep, kGateGrad, kStore, kStoreNarrow, kGradients };  // kStoreNarrow: no tile is wider than 128 columns
__host__ __device__ constexpr bool projects(Epilogue e) { return e == kGate || e == kGateKeep; }
__host__ __device__ constexpr bool stores(Epilogue e) { return e == kStore || e == kStoreNarrow; }

constexpr int kBlockK = 64;                       // elements of the contracted dimension in a stage
constexpr int kBoxBytes = 64 * 128;               // 64 lines of 64 16-bit elements
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (4 + kEpilogueWarps);
constexpr int kStageBuffer = 32 * 128;            // what a warp hands to the copy engine at once: 32 rows of 128 bytes
constexpr int kTile = 256;
constexpr int kTmemCols = 512;

template <Epilogue kEpi>
struct Shape {
  // Buffers of 4 KB for each storing warp, stages in what they leave.  Six stages instead of five: 8192 x 2048 x 4096 2 %, the
  // projections of 8192 x 5504 over 2048 4 %.
  static constexpr int kBuffers = kEpi == kGateGrad ? 4 : kEpi == kGateKeep ? 2 : 1;
  static constexpr int kBufferBytes = kEpilogueWarps * kBuffers * kStageBuffer;
  // A stage has 128 rows of A and 128 of B, 64 where tiles are narrow: eight stages then.  One round of narrow tiles is bound by the way from
  // L2, some 1.2 us for six or eight stages alike: 1856 tokens, 512 x 2048, both products 21.2 -> 20.4 us; 512 tokens, 1024 x 4096 28.5 -> 26.9.
  static constexpr int kStageBytes = (kEpi == kStoreNarrow ? 3 : 4) * kBoxBytes;
  static constexpr int kStages = kEpi == kGateGrad ? 3 : kEpi == kGateKeep ? 5 : kEpi == kStoreNarrow ? 8 : 6;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kBufferBytes;
  static_assert(kSmem + 1024 <= 232448, "shared memory");
};

struct Problem {
  CUtensorMap a, b;  // boxes of 64 lines
  CUtensorMap out;   // boxes of 32 lines (kGradients: fp32 or 16-bit elements)
  int m, n;
};

// Column sums of grad_y (rows, n_out) and of the (rows / 32, n_in) sums of the gradients of the pre-activations, each in kBands bands of
// rows, each band in the order of its rows: part[band] holds the n_in columns of the second, then those of the first.
constexpr int kBands = 296;
struct BiasSums {
  const void* grad_y;
  const float* sums;
  float* part;  // null: none wanted
  long long rows;
  int n_out, n_in;  // 0: not wanted
};

struct Params {
  Problem one;
  Problem two, input;       // kGradients: one and two are the weights', input the input's
  CUtensorMap b2;           // projections: the rows of the up projection, the odd CTA's
  CUtensorMap out2;         // kGateGrad: gradients of up
  CUtensorMap pre, pre2;    // pre-activations of gate | up (kGateKeep: written, boxes of 32 columns; kGateGrad: read); kGradients: pre = planes of partial sums
  const void* bias;         // projections: (2 n), kStore: (n); may be null
  uint2* exponents;         // of the pre-activations: (ceil(n / 64), m)
  float* column_sums;       // kGateGrad: (ceil(m / 32), 2 n) sums of the stored rows, or null
  int k;
  int whole, cut, tiles;    // tiles of full width, columns of a later one = full width / cut, pieces of work in all
  int slices;               // kStore: pieces of the contracted dimension, each with a plane (m, n) of partial sums in `pre`; 1: none
  // kGradients.  The weights' tiles: how many, the first, the first of the second product; in how many pieces their contracted dimension
  // is cut, and how many blocks a piece has.  The input's: its contracted dimension, and how many tiles the pairs without a weight tile
  // in the last round of those do meanwhile, each of them `ahead`; whole, cut and tiles are of the others.
  int weight_tiles, first, first2, pieces, per;
  int k_input, ahead, tiles_ahead;
  int wide_out;             // fp32 gradients of the weights
  BiasSums bias_sums;       // what the two idle warps of a CTA add meanwhile
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
// The default scope of the release, the CTA, is enough: what the arrival hands over is tensor memory, ordered by its own fences.  Released to
// the cluster, every arrival waited for the warp's stores: 1400 clocks of a tile's 4200 around the product.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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
__device__ __forceinline__ void umma_commit_own(uint64_t* bar) {  // in this CTA only
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
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

// kind::f16 with fp32 sums: D format (bits 4-5) 1 = f32, A (7-9) and B (10-12) 0 = f16, 1 = bf16; the columns go to bits 17-22
template <typename T, bool kAMn, bool kBMn>
__host__ __device__ constexpr uint32_t instruction() {
  constexpr uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)kAMn << 15) | ((uint32_t)kBMn << 16) | ((256u >> 4) << 24);
}

// Eight 16-bit values of a bias from column c on (a multiple of 8); zeros from column n on (n = 0: there is no bias).
template <typename T>
__device__ __forceinline__ uint4 bias8(const T* bias, int c, int n) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (c < n) v = *reinterpret_cast<const uint4*>(bias + c);
  return v;
}

// Where 16 bytes `chunk` of line `row` of a box lie.
__device__ __forceinline__ uint32_t box_chunk(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

// The same in a box of 32 columns, lines of 64 bytes (64-byte swizzle).
__device__ __forceinline__ uint32_t half_box_chunk(int row, int chunk) { return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)); }

// Column sums of a warp's buffer of 32 lines on mma.sync: the lines' transpose, 16 columns at a time, times ones.  Lane 4 i + j returns
// columns 16 j + i and 16 j + i + 8.  (As loads and additions they were a fifth of the instructions around the product.)
template <typename T>
__device__ __forceinline__ float2 column_sums32(uint32_t buffer, int lane) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const uint32_t one = kBf16 ? 0x3f803f80u : 0x3c003c00u;
  uint32_t a[4][2][4];
#pragma unroll
  for (int c = 0; c < 4; ++c)  // 16 columns
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // 16 lines; the four 8 x 8 parts: columns 0-7 | 8-15 of lines 0-7, then of lines 8-15
      const uint32_t at = buffer + box_chunk(16 * k + (lane & 7) + 8 * (lane >> 4), 2 * c + (lane >> 3 & 1));
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(a[c][k][0]), "=r"(a[c][k][1]), "=r"(a[c][k][2]), "=r"(a[c][k][3])
                   : "r"(at)
                   : "memory");
    }
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float d[4] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t(&m)[4] = a[c][k];
      if constexpr (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %8}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3]), "r"(one));
      else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %8}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3]), "r"(one));
    }
    if ((lane & 3) == c) sum = make_float2(d[0], d[2]);  // (all columns of the result are the same)
  }
  return sum;
}

template <typename T>
__device__ __forceinline__ void add8(float (&acc)[8], const T* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + 4);
    acc[0] += a.x, acc[1] += a.y, acc[2] += a.z, acc[3] += a.w, acc[4] += b.x, acc[5] += b.y, acc[6] += b.z, acc[7] += b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(x);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2<T>(w[e]);
      acc[2 * e] += f.x, acc[2 * e + 1] += f.y;
    }
  }
}
// One warp: a band of the rows of x (rows, n), n a multiple of 8.
template <typename T>
__device__ __forceinline__ void column_band(const T* x, long long rows, int n, int band, float* out, int lane) {
  const long long r0 = rows * band / kBands, r1 = rows * (band + 1) / kBands;
  for (int c = 8 * lane; c < n; c += 256) {
    float acc[8] = {};
    long long r = r0;
#pragma unroll 4
    for (; r < r1; ++r) add8(acc, x + r * n + c);
    reinterpret_cast<float4*>(out + c)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    reinterpret_cast<float4*>(out + c)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  }
}
template <typename T>
__device__ __forceinline__ void bias_band(const BiasSums& b, int band, int lane) {
  float* out = b.part + (size_t)band * (b.n_in + b.n_out);
  if (b.n_in) column_band(b.sums, (b.rows + 31) / 32, b.n_in, band, out, lane);
  if (b.n_out) column_band(static_cast<const T*>(b.grad_y), b.rows, b.n_out, band, out + b.n_in, lane);
}

// ---- the order of the work -----------------------------------------------------------------------------------------
// What a pair does at a time: `cols` columns from `col` of the rows from `row` on, over the blocks [k0, k1) of the contracted dimension.
enum Which { kOne, kTwo, kInput };
struct Work {
  int row, col, cols, k0, k1;
  Which which;  // kGradients
  int plane;    // where a part of a tile goes; -1: the whole
};

// Tiles are walked in groups of rows that stay in L2 together: all columns of kGroup row tiles, the row tiles fastest.
constexpr int kGroup = 8;
__host__ __device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int& m, int& n) {
  const int group = t / (kGroup * tiles_n), first = group * kGroup, rows = tiles_m - first < kGroup ? tiles_m - first : kGroup;
  t -= first * tiles_n;
  m = first + t % rows;
  n = t / rows;
}

template <Epilogue kEpi>
struct Walk {
  const Params& p;
  int pairs, k_blocks, tiles_m, tiles_n, t;
  int phase = 0, step = 0, place = 0, others = 0;  // kGradients
  __device__ Walk(const Params& q, int pair, int pairs_) : p(q), pairs(pairs_), t(pair) {
    k_blocks = (p.k + kBlockK - 1) / kBlockK;
    const Problem& tiled = kEpi == kGradients ? p.input : p.one;
    tiles_m = (tiled.m + kTile - 1) / kTile;
    tiles_n = (tiled.n + full() - 1) / full();
    if constexpr (kEpi == kGradients) {  // the pairs that have no tile in the last round of the weights' come first from then on
      const int last = p.weight_tiles * p.pieces % pairs;
      others = pairs - last;
      place = pair >= last ? pair - last : others + pair;
      step = place;
    }
  }
  __device__ static constexpr int full() { return projects(kEpi) ? kTile / 2 : kTile; }
  __device__ bool next(Work& w) {
    w.which = kOne, w.plane = -1, w.cols = full(), w.k0 = 0, w.k1 = k_blocks;
    if constexpr (kEpi == kGradients) {
      int m, n;
      if (phase == 0) {
        if (t < p.weight_tiles * p.pieces) {
          // The same piece of all tiles comes before the next piece of any: pairs that work at the same time read the same stretch of
          // the operands.  (Equal shares of all blocks in a row, where each pair is somewhere else, took 210 us instead of 100 on
          // 29 696 tokens: all operands came from memory again and again.)
          const int piece = t / p.weight_tiles, tile = p.first + t - piece * p.weight_tiles;
          w.k0 = piece * p.per, w.k1 = min(k_blocks, w.k0 + p.per);
          if (p.pieces > 1) w.plane = t;
          if (tile >= p.first2) {
            w.which = kTwo;
            tile_at(tile - p.first2, (p.two.m + kTile - 1) / kTile, (p.two.n + kTile - 1) / kTile, m, n);
          } else {
            tile_at(tile, (p.one.m + kTile - 1) / kTile, (p.one.n + kTile - 1) / kTile, m, n);
          }
          w.row = m * kTile, w.col = n * kTile;
          t += pairs;
          return true;
        }
        phase = 1;
      }
      w.which = kInput;
      w.k1 = (p.k_input + kBlockK - 1) / kBlockK;
      int tile, part = 0;
      if (phase == 1) {  // tiles that the others do ahead, row by row like the weights' tiles: what both read of [dg du] is in L2
        if (place < others && step < p.tiles_ahead && step < p.ahead * others) {
          tile = step;
          step += others;
          w.row = tile / tiles_n * kTile, w.col = tile % tiles_n * kTile;
          return true;
        }
        phase = 2, step = place;
      }
      if (step >= p.tiles) return false;
      if (step < p.whole) {
        tile = p.tiles_ahead + step;
      } else {
        tile = p.tiles_ahead + p.whole + (step - p.whole) / p.cut, part = (step - p.whole) % p.cut;
        w.cols = kTile / p.cut;
      }
      step += pairs;
      w.row = tile / tiles_n * kTile, w.col = tile % tiles_n * kTile + part * w.cols;
      return true;
    } else {
      const int slices = stores(kEpi) ? p.slices : 1;
      if (t >= p.tiles * slices) return false;
      int m, n, u = t;
      if (slices > 1) {
        const int per = (k_blocks + slices - 1) / slices;
        w.plane = t / p.tiles, u = t - w.plane * p.tiles;
        w.k0 = w.plane * per, w.k1 = min(k_blocks, w.k0 + per);
      }
      const bool whole = u < p.whole;
      const int part = whole ? 0 : (u - p.whole) % p.cut, tile = whole ? u : p.whole + (u - p.whole) / p.cut;
      if (!whole) w.cols = full() / p.cut;
      tile_at(tile, tiles_m, tiles_n, m, n);
      w.col = n * full() + part * w.cols;
      w.row = m * kTile;
      t += pairs;
      return true;
    }
  }
};

template <typename T, bool kAMn, bool kBMn, Epilogue kEpi, int kAct>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Params p) {
  using Sh = Shape<kEpi>;
  constexpr int kStages = Sh::kStages, kStageBytes = Sh::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ uint64_t bar_full[kStages], bar_empty[kStages], bar_acc[2], bar_drained[2], bar_in[2 * kEpilogueWarps], bar_end;
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    const int w = p.waits.withheld;
    for (int i = 0; i < kStages; ++i) mbar_init(&bar_full[i], 1 + (w == 0)), mbar_init(&bar_empty[i], 1 + (w == 1));
    for (int i = 0; i < 2; ++i) mbar_init(&bar_acc[i], 1 + (w == 2)), mbar_init(&bar_drained[i], 2 * kEpilogueWarps + (w == 3));
    for (int i = 0; i < 2 * kEpilogueWarps; ++i) mbar_init(&bar_in[i], 1);
    mbar_init(&bar_end, 1);
    mbar_fence_init();
  }
  if (warp == 2) {
    tmem_alloc2(&tmem_base_s, kTmemCols);
    tmem_relinquish2();
  }
  tc_fence_before_sync();
  cluster_sync();  // the barriers of both CTAs are ready
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;
  launch_dependents();
  wait_for_previous();

  Walk<kEpi> walk(p, pair, pairs);
  Work w;
  auto problem = [&](const Work& x) -> const Problem& { return kEpi == kGradients && x.which != kOne ? (x.which == kTwo ? p.two : p.input) : p.one; };
  bool bad = false;
  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (elect_one()) {
      uint32_t it = 0;
      while (!bad && walk.next(w)) {
        const Problem& prob = problem(w);
        const CUtensorMap* bmap = projects(kEpi) && rank ? &p.b2 : &prob.b;
        const bool outermost = kEpi == kGradients ? w.which != kInput : kAMn;  // the contracted dimension of A
        const int row = w.row + 128 * (int)rank;
        const int col = projects(kEpi) ? w.col : w.col + w.cols / 2 * (int)rank;
        const bool two = kEpi != kStoreNarrow && (projects(kEpi) ? w.cols : w.cols / 2) > 64;  // boxes of B (a tile of 64 columns uses half of its box)
        for (int kb = w.k0; kb < w.k1; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages && !mbar_wait_for(&bar_empty[s], ((it / kStages) & 1) ^ 1, p.waits.limit)) {
            bad = true;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&bar_full[s], 2 * (two ? 4 : 3) * kBoxBytes);
          const uint32_t bar = map_to_rank(smem_u32(&bar_full[s]), 0), dst = smem + s * kStageBytes;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            load_box2(dst + i * kBoxBytes, &prob.a, outermost ? row + 64 * i : kb * kBlockK, outermost ? kb * kBlockK : row + 64 * i, bar);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i == 0 || two)
              load_box2(dst + (2 + i) * kBoxBytes, bmap, kBMn ? col + 64 * i : kb * kBlockK, kBMn ? kb * kBlockK : col + 64 * i, bar);
        }
      }
      // The last products' arrivals on the stages of both CTAs are waited for as well: they come from the even CTA, and one that found the
      // odd one gone would write to whatever runs there next.
      if (!bad)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it && !bad; ++i)
          bad = !mbar_wait_for(&bar_empty[i % kStages], (i / kStages) & 1, p.waits.limit);
      if (bad && rank == 0) {  // copies that still fly write to these CTAs: their bytes arrive here (once a wait has lasted its second, all have)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
          if (!mbar_wait(&bar_full[i % kStages], (i / kStages) & 1)) break;
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---------------------------------------------------------------- products
    if (elect_one()) {
      // K-major: 16 elements of a line further on; MN-major: 16 lines further on, 64-wide chunks a box apart
      constexpr uint32_t kStepB = kBMn ? 16 * 128 : 32;
      const uint64_t b0 = make_smem_desc_sw128(smem + 2 * kBoxBytes, kBMn ? kBoxBytes : 0, 1024);
      uint32_t it = 0;
      for (int n = 0; !bad && walk.next(w); ++n) {
        const int buf = n & 1;
        if (n >= 2 && !mbar_wait_for(&bar_drained[buf], ((n >> 1) & 1) ^ 1, p.waits.limit)) {
          bad = true;
          break;
        }
        tc_fence_after_sync();
        const bool outermost = kEpi == kGradients ? w.which != kInput : kAMn;
        const uint32_t step_a = outermost ? 16 * 128 : 32;
        const uint64_t a0 = make_smem_desc_sw128(smem, outermost ? kBoxBytes : 0, 1024);
        const uint32_t idesc = (outermost ? instruction<T, true, kBMn>() : instruction<T, false, kBMn>()) | ((uint32_t)((projects(kEpi) ? 2 * w.cols : w.cols) >> 3) << 17);
        for (int kb = w.k0; kb < w.k1; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait_for(&bar_full[s], (it / kStages) & 1, p.waits.limit)) {
            bad = true;
            break;
          }
          tc_fence_after_sync();
          const uint64_t a = desc_advance(a0, s * kStageBytes), b = desc_advance(b0, s * kStageBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / 16; ++k)
            umma2(tmem + buf * kTile, desc_advance(a, k * step_a), desc_advance(b, k * kStepB), idesc, kb > w.k0 || k > 0);
          umma_commit2(&bar_empty[s]);
        }
        if (!bad) umma_commit2(&bar_acc[buf]);
      }
      if (bad) {  // no product may still run when the tensor memory is freed
        umma_commit_own(&bar_end);
        mbar_wait(&bar_end, 0);
      }
    }
  } else if (kEpi == kGradients && (warp == 2 || warp == 3)) {
    // ---------------------------------------------------------------- sums beside the products
    if (p.bias_sums.part)
      for (int band = 2 * blockIdx.x + warp - 2; band < kBands; band += 2 * gridDim.x) bias_band<T>(p.bias_sums, band, lane);
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- results
    const int ew = warp - 4, quad = warp & 3, half = ew >> 2;
    const uint32_t buffers = smem + kStages * kStageBytes + ew * Sh::kBuffers * kStageBuffer;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quad) << 16);
    const int lane_row = 128 * (int)rank + 32 * quad;
    uint32_t chunk = 0, fetched = 0;  // chunks of 64 columns (buffers handed over), counted over all tiles

    // a line of 64 16-bit columns of this lane's row, then the box
    auto put = [&](uint32_t dst, const uint32_t* words) {
#pragma unroll
      for (int v = 0; v < 8; ++v) sts128(dst + box_chunk(lane, v), make_uint4(words[4 * v], words[4 * v + 1], words[4 * v + 2], words[4 * v + 3]));
      fence_smem_to_async_proxy();
      __syncwarp();
    };
    auto emptied = [&]() {  // what this warp has handed over has left its buffers
      if (lane == 0) store_wait_read<0>();
      __syncwarp();
    };
    // Columns of a tile that this warp stores: half of them, all of them or none where they are a single chunk.
    auto mine = [&](const Work& x, int& first) {
      const int chunks = x.cols >= 128 ? x.cols / 128 : half == 0;
      first = half * (x.cols / 2);
      return chunks;
    };
    // kGateGrad: the pre-activations of 64 columns on their way to buffers 2 (i & 1) and 2 (i & 1) + 1
    auto fetch = [&](int col, int row) {
      const uint32_t i = fetched++;
      uint64_t* bar = &bar_in[2 * ew + (i & 1)];
      const uint32_t dst = buffers + 2 * (i & 1) * kStageBuffer;
      mbar_arrive_expect_tx(bar, 2 * kStageBuffer);
      load_box(dst, &p.pre, col, row, bar);
      load_box(dst + kStageBuffer, &p.pre2, col, row, bar);
    };
    Work later;  // kGateGrad: the tile after this one
    bool more = walk.next(later);
    if constexpr (kEpi == kGateGrad) {
      // a pair's later tiles are no wider: a warp with nothing to store in one has nothing in any after it
      int first;
      if (lane == 0 && more && mine(later, first)) fetch(later.col + first, later.row + lane_row);
    }
    uint2 exponents_next = make_uint2(0u, 0u);  // kGateGrad: of the chunk after this one
    auto exponents_at = [&](int col, int row) {
      uint2 v = make_uint2(0x0f0f0f0fu, 0x0f0f0f0fu);
      if (row < p.one.m && col < p.one.n) v = p.exponents[(size_t)(col >> 6) * p.one.m + row];
      return v;
    };
    if constexpr (kEpi == kGateGrad) {
      int first;
      if (more && mine(later, first)) exponents_next = exponents_at(later.col + first, later.row + lane_row + lane);
    }

    for (int n = 0; more; ++n) {
      w = later;
      more = walk.next(later);
      const int buf = n & 1, row0 = w.row + lane_row;
      int first;
      const int chunks = mine(w, first), col0 = w.col + first;
      const uint32_t acc = lane_base + buf * kTile;
      const T* bias = static_cast<const T*>(p.bias);
      const int bias_n = bias ? p.one.n : 0;
      uint4 bias_gate[2], bias_up[2];
      if constexpr (projects(kEpi)) {
#pragma unroll
        for (int v = 0; v < 2; ++v) bias_gate[v] = bias8(bias, col0 + 8 * v, bias_n), bias_up[v] = bias8(bias + bias_n, col0 + 8 * v, bias_n);
      }
      if (!mbar_wait_for(&bar_acc[buf], (n >> 1) & 1, p.waits.limit)) bad = true;
      bad = __any_sync(0xffffffffu, bad);
      if (bad) break;
      tc_fence_after_sync();
      auto drained = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_cluster(map_to_rank(smem_u32(&bar_drained[buf]), 0));
      };
      if (chunks == 0) drained();

      if constexpr (projects(kEpi)) {
        if (chunks) {  // 64 columns of gate and of up: hidden values in one buffer, the pre-activations of 32 columns at a time in the halves of the other
          uint32_t g[2][16], u[2][16];
          uint2 exponents = make_uint2(0u, 0u);
          const uint32_t keep = buffers + kStageBuffer;
          const bool stores = lane == 0 && row0 < p.one.m && col0 < p.one.n;
          tmem_ld16(acc + first, g[0]);
          tmem_ld16(acc + w.cols + first, u[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_wait();
            const uint4 bg[2] = {bias_gate[0], bias_gate[1]}, bu[2] = {bias_up[0], bias_up[1]};
            if (c < 3) {
              tmem_ld16(acc + first + 16 * (c + 1), g[(c + 1) & 1]);
              tmem_ld16(acc + w.cols + first + 16 * (c + 1), u[(c + 1) & 1]);
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                const int at = col0 + 16 * (c + 1) + 8 * v;
                bias_gate[v] = bias8(bias, at, bias_n), bias_up[v] = bias8(bias + bias_n, at, bias_n);
              }
            } else {
              drained();
            }
            uint32_t(&gv)[16] = g[c & 1], (&uv)[16] = u[c & 1], hw[8];
            PreGroup<T> of_gate, of_up;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const uint32_t bgw[4] = {bg[v].x, bg[v].y, bg[v].z, bg[v].w}, buw[4] = {bu[v].x, bu[v].y, bu[v].z, bu[v].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = 8 * v + 2 * e;
                const float2 gate = add2(make_float2(__uint_as_float(gv[i]), __uint_as_float(gv[i + 1])), unpack2<T>(bgw[e]));
                const float2 up = add2(make_float2(__uint_as_float(uv[i]), __uint_as_float(uv[i + 1])), unpack2<T>(buw[e]));
                const float2 h = mul2(activation2<kAct>(gate), up);
                hw[4 * v + e] = pack2<T>(h.x, h.y);
                if constexpr (kEpi == kGateKeep) {
                  gv[i] = __float_as_uint(gate.x), gv[i + 1] = __float_as_uint(gate.y), uv[i] = __float_as_uint(up.x), uv[i + 1] = __float_as_uint(up.y);
                  of_gate.add(gate.x, gate.y), of_up.add(up.x, up.y);
                }
              }
            }
            if (c == 0 || (kEpi == kGateKeep && c == 2)) emptied();  // (asked for after the arithmetic: it has had that long)
#pragma unroll
            for (int v = 0; v < 2; ++v) sts128(buffers + box_chunk(lane, 2 * c + v), make_uint4(hw[4 * v], hw[4 * v + 1], hw[4 * v + 2], hw[4 * v + 3]));
            if constexpr (kEpi == kGateKeep) {
              const uint32_t eg = of_gate.code(), eu = of_up.code();
              const PreForm<T> form_g(eg, false), form_u(eu, false);
              exponents.x |= eg << (8 * c), exponents.y |= eu << (8 * c);
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                uint32_t gw[4], uw[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int i = 8 * v + 2 * e;
                  gw[e] = form_g.pack(make_float2(__uint_as_float(gv[i]), __uint_as_float(gv[i + 1])));
                  uw[e] = form_u.pack(make_float2(__uint_as_float(uv[i]), __uint_as_float(uv[i + 1])));
                }
                const uint32_t at = keep + half_box_chunk(lane, 2 * (c & 1) + v);
                sts128(at, make_uint4(gw[0], gw[1], gw[2], gw[3]));
                sts128(at + kStageBuffer / 2, make_uint4(uw[0], uw[1], uw[2], uw[3]));
              }
            }
            if (c == 3 || (kEpi == kGateKeep && c == 1)) {
              fence_smem_to_async_proxy();
              __syncwarp();
              if (stores) {
                if (c == 3) store_box(&p.one.out, buffers, col0, row0);
                if (kEpi == kGateKeep && col0 + 16 * (c - 1) < p.one.n) {
                  store_box(&p.pre, keep, col0 + 16 * (c - 1), row0);
                  store_box(&p.pre2, keep + kStageBuffer / 2, col0 + 16 * (c - 1), row0);
                }
                store_commit();
              }
            }
          }
          if (kEpi == kGateKeep && row0 + lane < p.one.m && col0 < p.one.n) p.exponents[(size_t)(col0 >> 6) * p.one.m + row0 + lane] = exponents;
        }
      } else if constexpr (kEpi == kGateGrad) {
#pragma unroll 1
        for (int c = 0; c < chunks; ++c, ++chunk) {
          // the next chunk's pre-activations, once the buffers' previous results have left
          const bool last = c == chunks - 1;
          int f = 0;
          const uint2 exponents = exponents_next;
          if (!last || (more && mine(later, f))) {
            const int next_col = last ? later.col + f : col0 + 64 * (c + 1), next_row = last ? later.row + lane_row : row0;
            exponents_next = exponents_at(next_col, next_row + lane);
            if (lane == 0) {
              store_wait_read<0>();
              fetch(next_col, next_row);
            }
          }
          uint32_t d[2][16];
          tmem_ld16(acc + first + 64 * c, d[0]);
          if (!mbar_wait_for(&bar_in[2 * ew + (chunk & 1)], (chunk >> 1) & 1, p.waits.limit)) bad = true;
          bad = __any_sync(0xffffffffu, bad);
          if (bad) break;
          const uint32_t gate = buffers + 2 * (chunk & 1) * kStageBuffer, up = gate + kStageBuffer;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 gw[2], uw[2];
#pragma unroll
            for (int v = 0; v < 2; ++v) gw[v] = lds128(gate + box_chunk(lane, 2 * q + v)), uw[v] = lds128(up + box_chunk(lane, 2 * q + v));
            tmem_ld_wait();
            if (q < 3) tmem_ld16(acc + first + 64 * c + 16 * (q + 1), d[(q + 1) & 1]);
            else if (last) drained();
            const PreForm<T> form_g(exponents.x >> (8 * q) & 255u, true), form_u(exponents.y >> (8 * q) & 255u, true);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const uint32_t gs[4] = {gw[v].x, gw[v].y, gw[v].z, gw[v].w}, us[4] = {uw[v].x, uw[v].y, uw[v].z, uw[v].w};
              uint32_t dg[4], du[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 grad = make_float2(__uint_as_float(d[q & 1][8 * v + 2 * e]), __uint_as_float(d[q & 1][8 * v + 2 * e + 1]));
                float2 value, slope;
                activation2<kAct>(form_g.unpack(gs[e]), value, slope);
                const float2 a = mul2(mul2(grad, form_u.unpack(us[e])), slope), b = mul2(grad, value);
                dg[e] = pack2<T>(a.x, a.y), du[e] = pack2<T>(b.x, b.y);
              }
              sts128(gate + box_chunk(lane, 2 * q + v), make_uint4(dg[0], dg[1], dg[2], dg[3]));
              sts128(up + box_chunk(lane, 2 * q + v), make_uint4(du[0], du[1], du[2], du[3]));
            }
          }
          if (row0 + lane >= p.one.m) {  // rows beyond the last: zeros times an infinite weight are not zeros
#pragma unroll
            for (int v = 0; v < 8; ++v) sts128(gate + box_chunk(lane, v), make_uint4(0u, 0u, 0u, 0u)), sts128(up + box_chunk(lane, v), make_uint4(0u, 0u, 0u, 0u));
          }
          fence_smem_to_async_proxy();
          __syncwarp();
          const int col = col0 + 64 * c;
          if (lane == 0 && row0 < p.one.m && col < p.one.n) {
            store_box(&p.one.out, gate, col, row0);
            store_box(&p.out2, up, col, row0);
            store_commit();
          }
          if (p.column_sums && row0 < p.one.m) {  // of the values as stored
            const float2 dg = column_sums32<T>(gate, lane), du = column_sums32<T>(up, lane);
            const int at = col + 16 * (lane & 3) + (lane >> 2);
            float* to = p.column_sums + (size_t)(row0 >> 5) * (2 * (size_t)p.one.n) + at;
            if (at < p.one.n) to[0] = dg.x, to[p.one.n] = du.x;
            if (at + 8 < p.one.n) to[8] = dg.y, to[p.one.n + 8] = du.y;
            __syncwarp();
          }
        }
        if (bad) break;
      } else {
        const Problem& prob = problem(w);
        const bool sliced = stores(kEpi) && w.plane >= 0;
        if (sliced || (kEpi == kGradients && w.which != kInput && (w.plane >= 0 || p.wide_out))) {  // 32 fp32 columns at a time: partial sums, or an fp32 result
#pragma unroll 1
          for (int c = 0; c < 2 * chunks; ++c) {
            uint32_t d[32];
            tmem_ld32(acc + first + 32 * c, d);
            tmem_ld_wait();
            if (c == 2 * chunks - 1) drained();
            emptied();
            put(buffers, d);
            if (lane == 0 && row0 < prob.m && col0 + 32 * c < prob.n) {
              if (sliced) store_box3(&p.pre, buffers, col0 + 32 * c, row0, w.plane);
              else if (w.plane >= 0) store_box(&p.pre, buffers, first + 32 * c, w.plane * kTile + lane_row);
              else store_box(&prob.out, buffers, col0 + 32 * c, row0);
              store_commit();
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            uint32_t words[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t d[32];
              uint4 b[4];
              tmem_ld32(acc + first + 64 * c + 32 * h, d);
#pragma unroll
              for (int v = 0; v < 4; ++v) b[v] = stores(kEpi) ? bias8(bias, col0 + 64 * c + 32 * h + 8 * v, bias_n) : make_uint4(0u, 0u, 0u, 0u);
              tmem_ld_wait();
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const uint32_t bw[4] = {b[v].x, b[v].y, b[v].z, b[v].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 x = add2(make_float2(__uint_as_float(d[8 * v + 2 * e]), __uint_as_float(d[8 * v + 2 * e + 1])), unpack2<T>(bw[e]));
                  words[16 * h + 4 * v + e] = pack2<T>(x.x, x.y);
                }
              }
            }
            if (c == chunks - 1) drained();
            emptied();
            put(buffers, words);
            if (lane == 0 && row0 < prob.m && col0 + 64 * c < prob.n) {
              store_box(&prob.out, buffers, col0 + 64 * c, row0);
              store_commit();
            }
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
  if (bad) atomicExch(&g_gemm_status[p.waits.word], MF_ERR_DEVICE_TIMEOUT);
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();  // no arrival, copy or product of either CTA is outstanding
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc2(tmem, kTmemCols);
  }
}

}  // namespace gemm
}  // namespace mf
