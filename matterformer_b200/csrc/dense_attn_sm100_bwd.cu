// Dense attention with a learned bias by the offset on tcgen05, backward: head size 64 and 128, bf16 and fp16.  The probabilities are formed again.
//
// Two passes of one skeleton, a CTA owns a tile of 128 rows and walks over its partners in tiles of 64:
//   DQ  : owners = queries, partners = keys     S = Q K^T, dP = dO V^T       -> dS        -> dQ += dS K
//   DKV : owners = keys,    partners = queries  S^T = K Q^T, dP^T = V dO^T   -> P^T, dS^T -> dV += P^T dO, dK += dS^T Q
// Seven products instead of the five of a single pass, but every sum has one owner and a fixed order, and nothing is added up in memory.
// Two threads share a row, half of a step's columns each; P and dS are packed to 16 bits over the columns that S and dP had and are the A operands of the
// second products, whose sums stay in tensor memory over the whole walk.  Two groups of eight warps take the steps in turn, and S and dP have three
// buffers (two where the sums leave no room: DKV at head size 128), so that a group that is done with a step finds the next one ready: with a buffer for each group
// it waited for the second product of its step and the first ones of its next, and the pipes stood still (two cells of 4096 tokens 219 + 256 us).
//
// DKV wants the log-sum-exp and delta of the queries, its columns: they enter the products.  Each is three tf32 numbers, together as exact as fp32, in a further
// piece of the contracted dimension, whose other operand is ones, so that S and dP arrive with them subtracted (from shared memory they took a fifth of the pass).
//
// The bias of every offset up to the map's reach lies in shared memory (a few KB), so that a step reads it at its own place.  The table's gradient (DQ): steps whose offsets all fall into one bucket add up in a register; in the others dS goes through shared memory and threads sum
// along its diagonals, each into a column of sums of its own.  dS = P (dP - delta) with delta from rounded outputs; the row sums of dS, which are zero but for the error in
// delta, correct what far buckets got: there thousands of P share one error, which would otherwise be the largest of that sum.
//
// Two cells of 4096 tokens, 8 heads of 64, with the table's gradient: DQ 199 us (issue slots 53 %, tensor pipe 28 %: instructions and diagonals), DKV 166 us (tensor pipe
// 51 %); four causal sequences of 1024, 16 heads on 4 of 128: 61 + 63 us, start and end of short walks.
//
// Roles as in the forward kernel; the two warps that clear rows also bring the queries' log-sum-exp and delta for DKV.
#include "dense_attn_sm100.cuh"

namespace mf {
namespace {

__device__ int32_t g_dense_status[2];  // last expired wait: of calls, of the self-test
__device__ int32_t g_taken_status;
__global__ void take_status_kernel(int word) { g_taken_status = atomicExch(&g_dense_status[word], 0); }

constexpr int kOwnerWarps = 16, kBwdThreads = (kOwnerWarps + 4) * 32, kPart = 64, kCols = 32, kSpan = kTcRows + kPart - 1;
constexpr int kMostReach = 512;  // of the map, whose bias lies in shared memory
constexpr int kRegAux = 56, kRegOwner = 104;
static_assert(kOwnerWarps * kRegOwner + 4 * kRegAux <= (kOwnerWarps + 4) * 96, "register hand-over exceeds the CTA's pool");

template <int D, bool DKV, bool SUMS>
struct BwdShape {
  static constexpr int kChunks = D / 64, kTile = kChunks * kTcRows * 128, kPartTile = kChunks * kPart * 128;
  static constexpr int kBuffers = D == 128 && DKV ? 2 : 3, kColSums = 128 * kBuffers;
  static_assert(kColSums + (DKV ? 2 : 1) * D <= 512, "");
  static constexpr int kStages = D == 64 ? (SUMS ? 5 : 6) : SUMS || DKV ? 3 : 4;
  static constexpr int kOnes = DKV ? kTcRows * 128 : 0, kStatTile = DKV ? kPart * 128 : 0;  // lines of 128 bytes, of which 32 and 64 are used
  static constexpr int kOffA = 0, kOffB = kTile, kOffRing = 2 * kTile, kOffStats = kOffRing + kStages * 2 * kPartTile;
  static constexpr int kOffOnes = kOffStats + kStages * kStatTile, kSmem = kOffOnes + kOnes;
  static constexpr int kMostBuckets = D == 64 ? 64 : 32;  // whose sums fit beside that
  static constexpr int kDiagonals = D == 64 ? 16 : 8;     // columns of dS that 128 threads sum along their diagonals at a time
  static constexpr int kDiagonalBytes = kTcRows * (kDiagonals + 1) * 4;
};

// Diagonals of dS of the W columns from c0 + w0 on: offset of the diagonal that starts in row 127 - r (which = 0), or in column r + 1 (1, for r < W - 1 alone), among
// the kSpan of a step.  What other threads get for the latter is of no use to them, but an entry of the step all the same.
__host__ __device__ constexpr int diagonal_of(int which, int c0, int w0, int r) {
  const int e = c0 + w0 + r + (which ? kTcRows : 0);
  return e < kSpan ? e : kSpan - 1;
}
template <int W>
__host__ __device__ constexpr bool diagonals_fit() {  // entries of the step, and those that are used are the ones meant
  for (int c0 = 0; c0 < kPart; c0 += kCols)
    for (int w0 = 0; w0 < kCols; w0 += W)
      for (int r = 0; r < kTcRows; ++r)
        for (int which = 0; which < 2; ++which) {
          const int e = diagonal_of(which, c0, w0, r);
          if (e < 0 || e >= kSpan || ((which == 0 || r < W - 1) && e != c0 + w0 + r + which * kTcRows)) return false;
        }
  return true;
}

// D[tmem] += A[smem] * B[smem] of fp32 words, of which the tensor cores take the leading 11 bits of the mantissa; eight to an instruction
__device__ __forceinline__ void umma_tf32_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], da, db, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHiSw128)
      : "memory");
}
// a number as the sum of three that tf32 holds
__device__ __forceinline__ float4 three_parts(float v) {
  const float a = __uint_as_float(__float_as_uint(v) & 0xffffe000u), r = v - a;
  const float b = __uint_as_float(__float_as_uint(r) & 0xffffe000u);
  return make_float4(a, b, r - b, 0.f);
}

template <typename T, int D, bool DKV, bool TABLE>
__global__ void __launch_bounds__(kBwdThreads, 1) dense_attn_tc_bwd_kernel(const __grid_constant__ DenseTcParams tc) {
  using Sh = BwdShape<D, DKV, TABLE && !DKV>;
  constexpr int S = Sh::kStages, BUFFERS = Sh::kBuffers;
  const DenseParams& p = tc.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // behind the tiles: [2 groups][2 halves][128 rows][kDiagonals + 1] | [num_buckets][4 halves of groups][64] | bias of the offsets from -reach - kSpan + 1 to
  // reach + kSpan - 1 (DKV: for each group, they may be at different heads), their buckets
  const bool table_grad = TABLE && !DKV && p.dbias_part;
  const int offsets = TABLE ? 2 * p.reach + 2 * kSpan - 1 : 0;
  float* diagonals = reinterpret_cast<float*>(smem + Sh::kSmem);
  float* sums = reinterpret_cast<float*>(smem + Sh::kSmem + (table_grad ? 4 * Sh::kDiagonalBytes : 0));
  float* offset_bias = sums + (table_grad ? p.num_buckets * 256 : 0);
  uint8_t* offset_bucket = reinterpret_cast<uint8_t*>(offset_bias + (DKV ? 2 : 1) * offsets);
  __shared__ uint64_t bar_own, bar_full[S], bar_free[S], bar_clean[S], bar_s[BUFFERS], bar_p[BUFFERS], bar_o, bar_drain;
  __shared__ uint32_t tmem_base;
  __shared__ float errors[DKV ? 1 : 4][DKV ? 1 : 128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- which rows
  const int group = p.H / p.K, heads = DKV ? p.K : p.H, units = p.B * heads, tiles = gridDim.x / units;
  const int unit = p.causal ? blockIdx.x % units : blockIdx.x / tiles;
  const int tile_at = !p.causal ? blockIdx.x % tiles : DKV ? blockIdx.x / units : tiles - 1 - (int)(blockIdx.x / units);  // the longest walks first
  const int b = unit / heads, head = unit % heads, row0 = tile_at * kTcRows, kh = DKV ? head : head / group;
  const DenseLengths len = dense_lengths(p, b);
  const int own_rows = DKV ? len.nk : len.nq, own_all = DKV ? p.N : p.M;
  int from = 0, until = 0;  // partner steps of a head
  if (row0 < own_rows) {
    if (DKV) from = dense_first(p, len, row0) / kPart, until = (len.nq + kPart - 1) / kPart;
    else until = (dense_limit(p, len, min(row0 + kTcRows, len.nq) - 1) + kPart - 1) / kPart;
  }
  const int per_head = max(0, until - from), steps = DKV ? per_head * group : per_head;
  // A step's partners: row and head, moved on without divisions, which would be most of what some roles execute.
  struct Walk {
    int t, row, head;
  };
  auto begin = [&](int t) { return Walk{t, (from + (DKV ? t % per_head : t)) * kPart, DKV ? kh * group + t / per_head : kh}; };
  auto advance = [&](Walk& w, int by) {
    w.t += by, w.row += by * kPart;
    if (DKV)
      while (w.row >= until * kPart) w.row -= per_head * kPart, ++w.head;
  };
  auto first_offset = [&](int at) { return (DKV ? row0 - at - (kPart - 1) : at - row0 - (kTcRows - 1)) - len.shift; };  // of the pairs of a step
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.key_mask_batch : nullptr;
  const int part_rows = DKV ? len.nq : len.nk, part_all = DKV ? p.M : p.N;
  const bool cleaning = DKV || mask || part_rows < min(part_all, until * kPart);

  if (steps == 0) {
    if (tid < kTcRows && row0 + tid < own_all) {
      const int row = row0 + tid;
      auto clear = [&](void* base, const DenseRows& rows) {
        if (!base) return;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(base) + rows.at(b, head, row));
        for (int c = 0; c < D / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
      };
      if (DKV) {
        clear(p.dk, p.dk_rows);
        clear(p.dv, p.dv_rows);
      } else {
        clear(p.dq, p.dq_rows);
        p.delta[((long long)b * p.H + head) * p.M + row] = 0.f;
      }
    }
    if (TABLE && !DKV && p.dbias_part)
      for (int i = tid; i < p.num_buckets; i += kBwdThreads) p.dbias_part[((long long)unit * tiles + tile_at) * p.num_buckets + i] = 0.f;
    return;
  }

  if (tid == 0) {
    auto init = [&](uint64_t* bar, int count, int kind) { mbar_init(bar, count + (tc.waits.withheld == kind)); };
    init(&bar_own, 1, 0);
    for (int i = 0; i < S; ++i) init(&bar_full[i], 1, 0), init(&bar_free[i], 1, 1), init(&bar_clean[i], 2, 4);
    for (int x = 0; x < BUFFERS; ++x) init(&bar_s[x], 1, 2), init(&bar_p[x], 8, 3);
    init(&bar_o, 1, 2);
    mbar_init(&bar_drain, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base, 512);
    tmem_relinquish();
  }
  if (table_grad)
    for (int i = tid; i < p.num_buckets * 256; i += kBwdThreads) sums[i] = 0.f;
  if (TABLE && !DKV)
    for (int i = tid; i < offsets; i += kBwdThreads) {
      const int bucket = dense_offset_bucket(p, i - p.reach - (kSpan - 1));
      offset_bias[i] = dense_bias_entry(p, bucket, head);
      offset_bucket[i] = (uint8_t)bucket;
    }
  if (DKV) {
    for (int i = tid; i < Sh::kOnes / 16; i += kBwdThreads) {  // 1 1 1 0 in the first 16 bytes of a line
      const int r = i >> 3, chunk = (i & 7) ^ (r & 7);
      *reinterpret_cast<float4*>(smem + Sh::kOffOnes + i * 16) = chunk == 0 ? make_float4(1.f, 1.f, 1.f, 0.f) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = tid; i < S * Sh::kStatTile / 16; i += kBwdThreads) *reinterpret_cast<uint4*>(smem + Sh::kOffStats + i * 16) = make_uint4(0, 0, 0, 0);
    fence_smem_to_async_proxy();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base;
  bool bad = false;
  auto wait_on = [&](uint64_t* bar, uint32_t phase) {
    if (!bad) bad = !mbar_wait_for(bar, phase & 1, tc.waits.limit);
  };
  // columns: S and dP of buffer i at 128 i and 128 i + 64, then the sums
  auto col_sum = [&](int which) { return (uint32_t)(Sh::kColSums + D * which); };

  if (warp >= kOwnerWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegAux));
    if (warp == kOwnerWarps + 1) {
      // ---------------------------------------------------------------- copies
      if (lane == 0) {
        const CUtensorMap *own_a = DKV ? &tc.k : &tc.q, *own_b = DKV ? &tc.v : &tc.grad_out, *part_a = DKV ? &tc.q : &tc.k, *part_b = DKV ? &tc.grad_out : &tc.v;
        tma_prefetch_map(own_a);
        tma_prefetch_map(own_b);
        tma_prefetch_map(part_a);
        tma_prefetch_map(part_b);
        mbar_arrive_expect_tx(&bar_own, 2 * Sh::kTile);
        for (int c = 0; c < Sh::kChunks; ++c)
          for (int half = 0; half < 2; ++half) {  // (boxes have 64 rows)
            const uint32_t at = (c * kTcRows + half * 64) * 128;
            tma_box(smem_u32(smem + Sh::kOffA) + at, own_a, c * 64, row0 + half * 64, head, b, &bar_own);
            tma_box(smem_u32(smem + Sh::kOffB) + at, own_b, c * 64, row0 + half * 64, head, b, &bar_own);
          }
        Walk w = begin(0);
        for (; w.t < steps; advance(w, 1)) {
          const int stage = w.t % S;
          if (w.t >= S) wait_on(&bar_free[stage], w.t / S - 1);
          if (bad) break;
          mbar_arrive_expect_tx(&bar_full[stage], 2 * Sh::kPartTile);
          const uint32_t at = smem_u32(smem + Sh::kOffRing) + stage * 2 * Sh::kPartTile;
          for (int c = 0; c < Sh::kChunks; ++c) {
            tma_box(at + c * kPart * 128, part_a, c * 64, w.row, w.head, b, &bar_full[stage]);
            tma_box(at + Sh::kPartTile + c * kPart * 128, part_b, c * 64, w.row, w.head, b, &bar_full[stage]);
          }
        }
        const int t = w.t;
        // whoever gave up, no copy may be in flight when the CTA ends
        if (!mbar_wait_for(&bar_own, 0, tc.waits.limit)) bad = true;
        for (int i = max(0, t - S); i < t; ++i)
          if (!mbar_wait_for(&bar_full[i % S], (i / S) & 1, tc.waits.limit)) bad = true;
      }
    } else if (warp == kOwnerWarps) {
      // ---------------------------------------------------------------- products
      if (elect_one()) {
        const uint32_t l_a = make_desc_lo(smem_u32(smem + Sh::kOffA), 0), l_b = make_desc_lo(smem_u32(smem + Sh::kOffB), 0);
        const uint32_t l_ring = make_desc_lo(smem_u32(smem + Sh::kOffRing), 0), l_ring_mn = make_desc_lo(smem_u32(smem + Sh::kOffRing), kPart * 128);
        constexpr uint32_t kPartTile = Sh::kPartTile >> 4, kChunk = (kTcRows * 128) >> 4, kPartChunk = (kPart * 128) >> 4;
        const uint32_t l_ones = make_desc_lo(smem_u32(smem + Sh::kOffOnes), 0), l_stats = make_desc_lo(smem_u32(smem + Sh::kOffStats), 0);
        constexpr uint32_t idesc_stats = (make_idesc_bf16(kTcRows, kPart, false, false) & ~(0x3fu << 7)) | (2u << 7) | (2u << 10);  // tf32 by tf32
        constexpr uint32_t idesc_s = make_idesc_16<T>(kTcRows, kPart, false, false), idesc_o = make_idesc_16<T>(kTcRows, D, false, true);
        auto logits = [&](int t, int buffer) {
          const int stage = t % S;
          wait_on(cleaning ? &bar_clean[stage] : &bar_full[stage], t / S);
          tc_fence_after_sync();
          const uint32_t part = l_ring + stage * 2 * kPartTile, col = tmem + 128 * buffer;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            umma_ss_lo(col, l_a + (ks >> 2) * kChunk + (ks & 3) * 2, part + (ks >> 2) * kPartChunk + (ks & 3) * 2, idesc_s, ks > 0);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            umma_ss_lo(col + 64, l_b + (ks >> 2) * kChunk + (ks & 3) * 2, part + kPartTile + (ks >> 2) * kPartChunk + (ks & 3) * 2, idesc_s, ks > 0);
          if (DKV) {
            const uint32_t stat = l_stats + stage * (Sh::kStatTile >> 4);
            umma_tf32_lo(col, l_ones, stat, idesc_stats);
            umma_tf32_lo(col + 64, l_ones, stat + 2, idesc_stats);
          }
          umma_commit(&bar_s[buffer]);
        };
        wait_on(&bar_own, 0);
        for (int t = 0; t < min(BUFFERS, steps); ++t) logits(t, t);
#pragma unroll 1
        for (int t0 = 0; t0 < steps; t0 += BUFFERS) {
#pragma unroll
          for (int buffer = 0; buffer < BUFFERS; ++buffer) {
            const int t = t0 + buffer, stage = t % S;
            if (t >= steps) break;
            wait_on(&bar_p[buffer], t / BUFFERS);
            tc_fence_after_sync();
            const uint32_t part = l_ring_mn + stage * 2 * kPartTile, col = tmem + 128 * buffer;
#pragma unroll
            for (int kg = 0; kg < kPart / 16; ++kg) {
              const uint32_t packed = 32 * (kg >> 1) + 8 * (kg & 1);
              if (DKV) umma_ts_lo(tmem + col_sum(1), col + packed, part + kPartTile + 128 * kg, idesc_o, t > 0 || kg > 0);
              umma_ts_lo(tmem + col_sum(0), col + 64 + packed, part + 128 * kg, idesc_o, t > 0 || kg > 0);
            }
            umma_commit(&bar_free[stage]);
            if (t + BUFFERS < steps) logits(t + BUFFERS, buffer);
          }
        }
        umma_commit(&bar_o);
        // nor a product when tensor memory is given back
        umma_commit(&bar_drain);
        if (!mbar_wait(&bar_drain, 0)) bad = true;
      }
    } else {
      // ---------------------------------------------------------------- two warps, a row of the step for each lane: partners that are none become zeros;
      // log-sum-exp and delta of queries
      // (Both wait for every step: a warp that left steps out could meet a barrier two phases on and take it for its own.)
      if (cleaning) {
        const int c = lane + 32 * (warp - (kOwnerWarps + 2));
        int bias_head = -1;
        constexpr int AHEAD = DKV ? 3 : 1;
        float far_bias[2] = {0.f, 0.f}, lse[AHEAD], delta[AHEAD];
        const float per = 1.f / (p.scale * kDenseLog2e);
        Walk next = begin(0), w = next;  // of what is fetched, of what is put down
        auto fetch = [&](float& l, float& d) {  // steps ahead: one takes less time than its loads
          if (next.t >= steps) return;
          const int i = next.row + c;
          const long long stat = ((long long)b * p.H + next.head) * p.M + i;
          l = i < len.nq ? p.lse[stat] : INFINITY, d = i < len.nq ? p.delta[stat] : 0.f;  // (delta of a query that sees nothing is zero)
          advance(next, 1);
        };
        if (DKV)
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) fetch(lse[u], delta[u]);
        while (w.t < steps)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (w.t >= steps) break;
          const int stage = w.t % S, at = w.row;
          float one = 0.f;
          if (DKV && TABLE) {
            if (w.head != bias_head) {
              bias_head = w.head;
              far_bias[0] = dense_bias_entry(p, p.buckets[0], bias_head), far_bias[1] = dense_bias_entry(p, p.buckets[2 * p.reach], bias_head);
            }
            const int start = first_offset(at);
            one = start + kSpan - 1 <= -p.reach ? far_bias[0] : start >= p.reach ? far_bias[1] : 0.f;
          }
          const bool sees = lse[u] != INFINITY;  // queries that see nothing, and their gradients, may hold anything
          wait_on(&bar_full[stage], w.t / S);
          if (DKV) {
            float v = (one - lse[u]) * fabsf(per);
            if (v < -1e30f) v = -1e30f;  // p = 0 (a number: the parts of an infinity are none)
            uint8_t* line = smem + Sh::kOffStats + stage * Sh::kStatTile + c * 128;
            *reinterpret_cast<float4*>(line + ((0 ^ (c & 7)) << 4)) = three_parts(per < 0.f ? -v : v);
            *reinterpret_cast<float4*>(line + ((2 ^ (c & 7)) << 4)) = three_parts(-delta[u]);
          }
          const bool there = at + c < part_rows && (DKV ? sees : !mask || mask[at + c]);
          if (!bad && !there && at + c < part_all) {  // (what lies behind the tensor is zeros already)
#pragma unroll 1
            for (int i = 0; i < 2 * Sh::kChunks * 8; ++i)
              *reinterpret_cast<uint4*>(smem + Sh::kOffRing + (stage * 2 * Sh::kChunks + i / 8) * kPart * 128 + c * 128 + (i % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_smem_to_async_proxy();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_clean[stage]);
          if (DKV) fetch(lse[u], delta[u]);
          advance(w, 1);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ row owners
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegOwner));
    const int y = warp >> 3, half = warp >> 2 & 1, r = tid & 127;  // group, half of the columns, row
    const int c0 = half * kCols, pair = tid & 255, team = warp >> 2;  // the 256 threads of a group are pairs of 128
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int row = row0 + r;
    bool row_ok = row < own_rows;
    const float sc2 = p.scale * kDenseLog2e;
    float lse = 0.f, delta = 0.f;
    // visible partners of this row: [lo, hi) at DKV and DQ; a row that is none may see what it wants
    int lo = INT32_MIN, hi = INT32_MAX;
    if (!DKV) {
      const long long stat = ((long long)b * p.H + head) * p.M;
      if (row_ok) {
        hi = dense_limit(p, len, row);
        lse = p.lse[stat + row];
        row_ok = lse != INFINITY;  // a query that sees nothing, and its gradient, may hold anything
        // delta: a quarter of the channels each
        const uint4* go = reinterpret_cast<const uint4*>(static_cast<const T*>(p.grad_out) + p.go_rows.at(b, head, row) + team * (D / 4));
        const uint4* o = reinterpret_cast<const uint4*>(static_cast<const T*>(p.out) + p.out_rows.at(b, head, row) + team * (D / 4));
        uint4 u[D / 32], w[D / 32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) u[c] = go[c], w[c] = o[c];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint32_t uw[4] = {u[c].x, u[c].y, u[c].z, u[c].w}, ww[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2<T>(uw[e]), g = unpack2<T>(ww[e]);
            delta = fmaf(f.x, g.x, fmaf(f.y, g.y, delta));
          }
        }
      }
      errors[team][r] = delta;
      group_barrier(7, 512);
      delta = (errors[0][r] + errors[1][r]) + (errors[2][r] + errors[3][r]);
      if (!row_ok) delta = 0.f;
      if (row < p.M && team == 0) p.delta[stat + row] = delta;
    } else if (row_ok) {
      lo = dense_first(p, len, row);
    }
    const int tile_lo = __reduce_max_sync(0xffffffffu, lo), tile_hi = __reduce_min_sync(0xffffffffu, hi);
    float far[2] = {0.f, 0.f}, far_p[2] = {0.f, 0.f}, all = 0.f;  // sums of dS and of P over steps of one bucket (offsets below, above), of dS over all
    int bias_head = -1;
    const float* const my_bias = offset_bias + (DKV ? y * offsets : 0);
    Walk w = begin(min(y, steps - 1));
    int buffer = y, phase = 0;  // step w.t is the phase-th of its buffer
    for (w.t = y; w.t < steps; advance(w, 2)) {
      const int at = w.row;
      const uint32_t col = tmem + lanes + 128 * buffer;
      float one = 0.f;
      const float* near = nullptr;  // bias of the thread's column c at near[c] (DQ), near[-c] (DKV)
      const uint8_t* near_bucket = nullptr;
      int side = 0;
      if (TABLE) {
        const int start = first_offset(at);  // entry e: the offset start + e
        if (DKV && w.head != bias_head) {
          if (bias_head >= 0) group_barrier(1 + y, 256);
          bias_head = w.head;
          for (int i = pair; i < offsets; i += 256)
            offset_bias[y * offsets + i] = dense_bias_entry(p, dense_offset_bucket(p, i - p.reach - (kSpan - 1)), bias_head);
          group_barrier(1 + y, 256);
        }
        if (start + kSpan - 1 <= -p.reach || start >= p.reach) {
          side = start >= p.reach;
          if (!DKV) one = my_bias[side ? offsets - 1 : 0];  // (DKV: with the log-sum-exp)
        } else {
          const int entry = start + p.reach + kSpan - 1;
          near = my_bias + entry + (DKV ? r + kPart - 1 - c0 : kTcRows - 1 - r + c0);
          near_bucket = offset_bucket + entry;
        }
      }
      uint32_t seen = ~0u;
      if (!DKV && mask) {
        const int key = at + c0 + lane;
        seen = __ballot_sync(0xffffffffu, key < len.nk && mask[key] != 0);
      }
      wait_on(&bar_s[buffer], phase);
      tc_fence_after_sync();
      float z[kCols], d[kCols];
      tmem_ld32(col + c0, *reinterpret_cast<uint32_t(*)[32]>(&z[0]));
      tmem_ld32(col + 64 + c0, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
      tmem_ld_wait();
      auto form = [&](auto biased) {  // p into z, dP - delta into d
        constexpr bool kBiased = decltype(biased)::value;
        const float2 less = make_float2(one - lse, one - lse), off = make_float2(-delta, -delta), by = make_float2(sc2, sc2);
#pragma unroll
        for (int c = 0; c < kCols; c += 2) {
          const float2 q = make_float2(z[c], z[c + 1]);
          float2 e;
          if constexpr (DKV && !kBiased) e = mul2(q, by);
          else if constexpr (DKV) e = fma2(q, by, make_float2(near[-c], near[-c - 1]));
          else if constexpr (kBiased) e = fma2(q, by, add2(less, make_float2(near[c], near[c + 1])));
          else e = fma2(q, by, less);
          z[c] = dense_exp2(e.x), z[c + 1] = dense_exp2(e.y);
          if constexpr (!DKV) {
            const float2 v = add2(make_float2(d[c], d[c + 1]), off);
            d[c] = v.x, d[c + 1] = v.y;
          }
        }
      };
      if (TABLE && near) form(std::true_type{});
      else form(std::false_type{});
      if (at < tile_lo || at + kPart > tile_hi || (!DKV && mask)) {
        const int a = lo == INT32_MIN ? -1 : lo - at - c0, e = hi == INT32_MAX ? kPart : hi - at - c0;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          if (c < a || c >= e || !((seen >> c) & 1u)) z[c] = 0.f;
      }
      uint32_t packed[16];
      if (DKV) {
#pragma unroll
        for (int c = 0; c < kCols; c += 2) packed[c >> 1] = pack2<T>(z[c], z[c + 1]);
        tmem_st16(col + c0, packed);  // (over the thread's own columns: the other half may not have read its)
      }
#pragma unroll
      for (int c = 0; c < kCols; c += 2) {
        const float2 v = mul2(make_float2(z[c], z[c + 1]), make_float2(d[c], d[c + 1]));
        d[c] = v.x, d[c + 1] = v.y;
        packed[c >> 1] = pack2<T>(v.x, v.y);
      }
      tmem_st16(col + 64 + c0, packed);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[buffer]);
      buffer += 2;
      if (buffer >= BUFFERS) buffer -= BUFFERS, ++phase;
      if (table_grad) {
        float2 u[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kCols; c += 2) u[(c >> 1) & 1] = add2(u[(c >> 1) & 1], make_float2(d[c], d[c + 1]));
        const float sum = (u[0].x + u[0].y) + (u[1].x + u[1].y);
        all += sum;
        if (near) {
          // Pairs of one offset lie on a diagonal: a thread adds up one or two of them, which have one bucket each.  Threads 64 apart share a column
          // of sums and take it in turn.
          constexpr int W = Sh::kDiagonals;
          float* tile = diagonals + team * kTcRows * (W + 1);
          float* column = sums + team * 64 + (r & 63);
#pragma unroll
          for (int w0 = 0; w0 < kCols; w0 += W) {
#pragma unroll
            for (int c = 0; c < W; ++c) tile[r * (W + 1) + c] = row_ok ? d[w0 + c] : 0.f;
            group_barrier(3 + team, 128);
            float v[2] = {0.f, 0.f};  // c - row = r - 127 and r + 1
            const int row_at = kTcRows - 1 - r;
#pragma unroll
            for (int c = 0; c < W; ++c)
              if (row_at + c < kTcRows) v[0] += tile[(row_at + c) * (W + 1) + c];
            if (r < W - 1) {
#pragma unroll
              for (int c = 1; c < W; ++c)
                if (c > r) v[1] += tile[(c - r - 1) * (W + 1) + c];
            }
            static_assert(diagonals_fit<W>(), "a step has the buckets of kSpan offsets");
            const int b0 = near_bucket[diagonal_of(0, c0, w0, r)], b1 = near_bucket[diagonal_of(1, c0, w0, r)];
            if (r < 64) {
              if (b0 < p.num_buckets) column[b0 * 256] += v[0];
              if (r < W - 1 && b1 < p.num_buckets) column[b1 * 256] += v[1];
            }
            group_barrier(3 + team, 128);
            if (r >= 64 && b0 < p.num_buckets) column[b0 * 256] += v[0];
          }
        } else {
          float2 v[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < kCols; c += 2) v[(c >> 1) & 1] = add2(v[(c >> 1) & 1], make_float2(z[c], z[c + 1]));
          far[0] += side ? 0.f : sum, far[1] += side ? sum : 0.f;
          const float mass = (v[0].x + v[0].y) + (v[1].x + v[1].y);
          far_p[0] += side ? 0.f : mass, far_p[1] += side ? mass : 0.f;
        }
      }
    }
    if (table_grad) {
      group_barrier(7, 512);  // a group without a step is here while the other may still read its delta
      errors[team][r] = all;  // four threads worked on the row
      group_barrier(7, 512);
      all = (errors[0][r] + errors[1][r]) + (errors[2][r] + errors[3][r]);
      float* column = sums + team * 64 + (r & 63);
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        if ((r >= 64) == (turn == 1)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int bucket = p.buckets[e ? 2 * p.reach : 0];
            if (bucket < p.num_buckets && row_ok) column[bucket * 256] += far[e] - all * far_p[e];
          }
        }
        group_barrier(7, 512);
      }
      float* part = p.dbias_part + ((long long)unit * tiles + tile_at) * p.num_buckets;
      for (int i = warp; i < p.num_buckets; i += kOwnerWarps) {
        float v = 0.f;
        for (int e = lane; e < 256; e += 32) v += sums[i * 256 + e];
        v = warp_sum(v);
        if (lane == 0) part[i] = v;
      }
    }

    // ---- rows out: zeros for what is no row
    wait_on(&bar_o, 0);
    tc_fence_after_sync();
    const bool real = row_ok && (!DKV || !mask || mask[row]);
    auto rows_out = [&](void* base, const DenseRows& rows, int which, int c0, int c1, float mul) {
#pragma unroll 1
      for (int c = c0; c < c1; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem + lanes + col_sum(which) + c, o);
        tmem_ld_wait();
        if (base && row < own_all) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(base) + rows.at(b, head, row) + c);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = real ? pack2<T>(__uint_as_float(o[e + 2 * i]) * mul, __uint_as_float(o[e + 2 * i + 1]) * mul) : 0u;
            dst[e >> 3] = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    };
    if (DKV) {  // a group for each gradient
      if (y == 0) rows_out(p.dk, p.dk_rows, 0, half * (D / 2), (half + 1) * (D / 2), p.scale);
      else rows_out(p.dv, p.dv_rows, 1, half * (D / 2), (half + 1) * (D / 2), 1.f);
    } else if (D == 128 || half == 0) {  // a quarter of the channels for 128 threads, or a half
      constexpr int share = 32;
      const int first_channel = (D == 128 ? team : y) * share;
      rows_out(p.dq, p.dq_rows, 0, first_channel, first_channel + share, p.scale);
    }
    tc_fence_before_sync();
  }
  if (bad) atomicExch(&g_dense_status[tc.waits.word], MF_ERR_DEVICE_TIMEOUT);
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <typename T, int D, bool DKV, bool TABLE>
int launch(const DenseTcParams& tc, cudaStream_t stream) {
  const DenseParams& p = tc.p;
  using Sh = BwdShape<D, DKV, TABLE && !DKV>;
  constexpr auto kernel = dense_attn_tc_bwd_kernel<T, D, DKV, TABLE>;
  auto offset_bytes = [](int reach) { return (2 * reach + 2 * kSpan - 1) * (DKV ? 2 * 4 : 4 + 1); };
  constexpr int most = Sh::kSmem + 1024 + (TABLE && !DKV ? 4 * Sh::kDiagonalBytes + Sh::kMostBuckets * 1024 : 0) + (TABLE ? (2 * kMostReach + 2 * kSpan - 1) * 8 : 0);
  static_assert(most <= 227 * 1024 - (DKV ? 512 : 2560), "beside the static part");
  const int smem = Sh::kSmem + 1024 + (TABLE && !DKV && p.dbias_part ? 4 * Sh::kDiagonalBytes + p.num_buckets * 1024 : 0) + (TABLE ? offset_bytes(p.reach) : 0);
  const cudaError_t err = allow_shared<dense_attn_tc_bwd_kernel<T, D, DKV, TABLE>>(most);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  const long long blocks = (long long)(((DKV ? p.N : p.M) + kTcRows - 1) / kTcRows) * p.B * (DKV ? p.K : p.H);
  kernel<<<(unsigned)blocks, kBwdThreads, smem, stream>>>(tc);
  MF_CHECK_LAUNCH("dense attention backward on tcgen05");
  return MF_OK;
}

template <typename T, int D>
int pick(const DenseTcParams& tc, bool table, cudaStream_t stream) {
  const int rc = table ? launch<T, D, false, true>(tc, stream) : launch<T, D, false, false>(tc, stream);
  if (rc != MF_OK || (!tc.p.dk && !tc.p.dv)) return rc;
  return table ? launch<T, D, true, true>(tc, stream) : launch<T, D, true, false>(tc, stream);
}

}  // namespace

int dense_attn_take_bwd_status(int word, int32_t* host_status, cudaStream_t stream) {
  take_status_kernel<<<1, 1, 0, stream>>>(word);
  MF_CHECK_LAUNCH("dense attention status read-back");
  cudaError_t e = cudaMemcpyFromSymbolAsync(host_status, g_taken_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "dense attention status read-back");
}

bool dense_tc_bwd_takes(const DenseParams& p, int head_dim, int kind, bool table_grad) {
  if (kind == MF_BUCKETS_PAIR || !dense_tc_takes(p, head_dim, kind)) return false;
  if (!(fabsf(p.scale) >= 1e-6f && fabsf(p.scale) <= 1e6f)) return false;  // (the log-sum-exp is divided by it)
  return kind == MF_BUCKETS_NONE || (p.reach <= kMostReach && (!table_grad || p.num_buckets <= (head_dim == 64 ? 64 : 32)));
}

int dense_attn_sm100_bwd(const DenseTcParams& tc, int dtype, int head_dim, int kind, cudaStream_t stream) {
  const bool table = kind != MF_BUCKETS_NONE;
  if (head_dim == 64) return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, 64>(tc, table, stream) : pick<__half, 64>(tc, table, stream);
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, 128>(tc, table, stream) : pick<__half, 128>(tc, table, stream);
}

}  // namespace mf
