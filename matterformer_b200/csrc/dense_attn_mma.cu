// Dense attention with a learned bias by buckets on the warp-level tensor cores (mma.sync m16n8k16): any length, head size 32, 64 or 128,
// any mask.
//
// One CTA of four warps owns 64 rows of one (batch, head), a warp 16 of them, and walks over tiles of 64 partner rows that arrive by cp.async
// while the previous tile is worked on.
//   FWD : owners = queries, partners = keys     out, lse      (running maximum and sum per row)
//   DQ  : owners = queries, partners = keys     dq, delta and the table's gradient per bucket
//   DKV : owners = keys,    partners = queries of all heads that share them     dk, dv  (logits formed transposed)
// Logits, probabilities and their gradients stay in registers: the C fragment of a product is the A operand of the next.  P and dS are
// rounded to the operands' type there (half a unit of 2^-8 or 2^-11 each, on terms of a sum), the only type the tensor cores take.
// Every output has one owner and a fixed order of its sums.
//
// Registers bound it: 64 x 64 logits, their gradients and the sums are 128 to 168 of a thread's, three or four CTAs on an SM (without that limit 255 and two, 64
// molecules of 19 to 192 tokens 124 us instead of 120 for forward and backward, 116 now), which use a third of the issue slots and a fifth of the tensor pipe. There: forward 26,
// DQ 48, DKV 39 us; 8 x 577 fp16 queries on 1000 keys, 4 heads of 32, 22 + 26 + 19 us. 64 rows to a tile: fewer waste products for molecules of all lengths.
#include "dense_attn.cuh"

namespace mf {
namespace {

enum { D_FWD = 0, D_DQ = 1, D_DKV = 2 };
constexpr int kOwn = 64, kPart = 64, kThreads = 128;
constexpr int kSpan = kOwn + kPart - 1;  // offsets between the rows of two tiles

template <int D>
constexpr int kTileBytes = 64 * (D + 8) * 2;

// Buffers of partner tiles.  Backward at head size 128 one: with two, 120 KB, an SM has room for one CTA, while of two CTAs one brings its tile as the other
// works (forward and backward, by pairs, one | two buffers: 731 x 54 tokens, 4 heads on 1, 238 | 351 us; 64 x 192 tokens, 8 heads, 273 | 366; 2 x 2171 queries on 6439 keys,
// one head, 702 | 759).  The queries' gradient by pairs too, for a third CTA beside up to 64 buckets' sums: 64 x 192 tokens, 8 heads of 64, 142 | 155 us.
template <int D, int MODE, int KIND>
constexpr int kStages = (D == 128 && MODE != D_FWD) || (MODE == D_DQ && KIND == MF_BUCKETS_PAIR) ? 1 : 2;
// shared memory: own_a | own_b (backward) | part_a[S] | part_b[S] | lse, delta [S][64] each (DKV) | table[kTableEntries] (pairs) | bias of offsets [S][128], their
// buckets [S][128] (offsets) | pairs' buckets [S][64][80] | DQ with a table: [4 warps][num_buckets + 1][32]
constexpr int kPairRow = 80, kPairTile = 64 * kPairRow;  // a row of 64 bytes, in banks of its own among eight neighbours
template <int D, int MODE, int KIND>
struct Layout {
  static constexpr int kS = kStages<D, MODE, KIND>;
  static constexpr int kStats = ((MODE == D_FWD ? 1 : 2) + 2 * kS) * kTileBytes<D>, kTable = kStats + (MODE == D_DKV ? kS * 2 * 64 * 4 : 0);
  static constexpr int kOffsets = kTable + (KIND == MF_BUCKETS_PAIR ? kTableEntries * 4 : 0), kPairs = kOffsets + (KIND == MF_BUCKETS_OFFSET ? kS * 128 * 5 : 0);
  static constexpr int kFixed = kPairs + (KIND == MF_BUCKETS_PAIR ? kS * kPairTile : 0);
};

// bits lo .. hi - 1 of a word
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  const uint32_t below = hi >= 32 ? ~0u : hi > 0 ? (1u << hi) - 1u : 0u, from = lo >= 32 ? 0u : lo > 0 ? ~0u << lo : ~0u;
  return below & from;
}

// rows [row0, row0 + 64) of a head, zeros from row_limit on and where `shown` (a bit for each) says so
template <typename T, int D>
__device__ __forceinline__ void load_rows(uint32_t tile, const T* src, long long stride, int row0, int row_limit, uint2 shown) {
  constexpr int LD = D + 8, PER_ROW = D / 8;
#pragma unroll
  for (int it = 0; it < 64 * PER_ROW / kThreads; ++it) {
    const int idx = it * kThreads + threadIdx.x;
    const int r = idx / PER_ROW, c = idx % PER_ROW, row = row0 + r;
    const bool ok = row < row_limit && (((r & 32 ? shown.y : shown.x) >> (r & 31)) & 1u);
    cp_async16(tile + (r * LD + c * 8) * 2, src + (ok ? row * stride : 0) + c * 8, ok);
  }
}

template <typename T, int D, int MODE, int KIND>
__global__ void __launch_bounds__(kThreads, D <= 64 ? (MODE == D_FWD ? 4 : 3) : 2) dense_attn_mma_kernel(const __grid_constant__ DenseParams p) {
  constexpr int LD = D + 8, TILE = kTileBytes<D>, KS = D / 16, STAGES = kStages<D, MODE, KIND>;
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t s_own_a = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), s_own_b = s_own_a + TILE;
  const uint32_t s_part_a = MODE == D_FWD ? s_own_b : s_own_b + TILE, s_part_b = s_part_a + STAGES * TILE;
  using At = Layout<D, MODE, KIND>;
  float* part_lse = reinterpret_cast<float*>(smem + At::kStats);
  float* part_delta = part_lse + STAGES * 64;
  float* table = reinterpret_cast<float*>(smem + At::kTable);
  float* offset_bias = reinterpret_cast<float*>(smem + At::kOffsets);
  uint8_t* offset_bucket = reinterpret_cast<uint8_t*>(offset_bias + STAGES * 128);
  uint8_t* pair_tile = smem + At::kPairs;
  float* sums = reinterpret_cast<float*>(smem + At::kFixed);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int heads = MODE == D_DKV ? p.K : p.H, group = p.H / p.K;
  // DQ with a table: CTAs stay with a head and take every slots-th of its tiles, so that the table's column is laid out and its sums are added up once for
  // all of them; a tile of a small molecule takes less time than that.  Otherwise a tile each, the longest walks of a causal call first.
  constexpr bool STAY = MODE == D_DQ && KIND != MF_BUCKETS_NONE;
  const int entries = p.B * heads, tiles = ((MODE == D_DKV ? p.N : p.M) + kOwn - 1) / kOwn, slots = STAY ? gridDim.x / heads : 1;
  const int nb = p.num_buckets;
  float* my_sums = sums + (warp * (nb + 1)) * 32 + lane;
  if (STAY) {
    if (KIND == MF_BUCKETS_PAIR)
      for (int i = tid; i < kTableEntries; i += kThreads) table[i] = dense_bias_entry(p, i, blockIdx.x % heads);
    if (p.dbias_part)
      for (int i = tid; i < 4 * (nb + 1) * 32; i += kThreads) sums[i] = 0.f;
  }
  for (int item = STAY ? blockIdx.x / heads : 0; item < (STAY ? p.B * tiles : 1); item += slots) {
  const int place = STAY ? item * heads + (int)(blockIdx.x % heads) : (int)blockIdx.x;
  int tile, b, oh;  // oh: head of the owners
  if (STAY) {
    b = item / tiles, tile = item % tiles, oh = place % heads;
  } else {
    const int entry = p.causal ? place % entries : place / tiles;
    tile = !p.causal ? place % tiles : MODE == D_DKV ? place / entries : tiles - 1 - place / entries;
    b = entry / heads, oh = entry % heads;
  }
  const int kh = MODE == D_DKV ? oh : oh / group;
  const DenseLengths len = dense_lengths(p, b);
  const int row0 = tile * kOwn;
  const int my = row0 + warp * 16 + g;  // this thread's rows: my, my + 8
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.key_mask_batch : nullptr;

  // ---- what the tile walks over: partners [first, last) in tiles, for DKV once for each head of the group
  const int own_limit = MODE == D_DKV ? len.nk : len.nq;
  int first = 0, last = 0;
  if (row0 < own_limit) {
    if (MODE == D_DKV) first = dense_first(p, len, row0) / kPart * kPart, last = len.nq;
    else last = dense_limit(p, len, min(row0 + kOwn, len.nq) - 1);
  }
  const int per_head = last > first ? (last - first + kPart - 1) / kPart : 0;
  const int steps = MODE == D_DKV ? per_head * group : per_head;

  const T* K = static_cast<const T*>(p.k) + p.k_rows.at(b, kh, 0);
  const T* V = static_cast<const T*>(p.v) + p.v_rows.at(b, kh, 0);
  auto q_of = [&](int h) { return static_cast<const T*>(p.q) + p.q_rows.at(b, h, 0); };
  auto go_of = [&](int h) { return static_cast<const T*>(p.grad_out) + p.go_rows.at(b, h, 0); };
  auto stat = [&](int h) { return ((long long)b * p.H + h) * p.M; };

  const bool aligned = KIND == MF_BUCKETS_PAIR && !((reinterpret_cast<uintptr_t>(p.buckets) | p.bucket_row | p.bucket_batch) & 15);
  // the buckets of 64 queries from i0 on and 64 keys from j0 on, zeros where there are none
  auto load_pairs = [&](int i0, int j0, int stage) {
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int idx = it * kThreads + tid, r = idx >> 2, c = (idx & 3) * 16;
      const bool ok = i0 + r < len.nq && j0 + c < len.nk;
      const uint8_t* src = p.buckets + (ok ? b * p.bucket_batch + (i0 + r) * p.bucket_row + j0 + c : 0);
      uint8_t* dst = pair_tile + stage * kPairTile + r * kPairRow + c;
      const int n = ok ? p.N - j0 - c : 0;  // (a row's storage may end with its last key, whatever the stride)
      if (aligned) {
        cp_async_part16(static_cast<uint32_t>(__cvta_generic_to_shared(dst)), src, min(n, 16));
      } else {
        const uint2 x = eight_bytes(src, n), y = eight_bytes(src + 8, n - 8);
        *reinterpret_cast<uint4*>(dst) = make_uint4(x.x, x.y, y.x, y.y);
      }
    }
  };
  // The key mask of 64 keys from j0 on: a byte for each lane and half, as bits.  They are asked for a tile before the rows are, which wait for them.
  auto mask_bytes = [&](int j0) {
    const int j = j0 + lane;
    return make_uchar2(j < len.nk ? mask[j] : 0, j + 32 < len.nk ? mask[j + 32] : 0);
  };
  auto mask_bits = [&](uchar2 m) { return make_uint2(__ballot_sync(0xffffffffu, m.x != 0), __ballot_sync(0xffffffffu, m.y != 0)); };
  const uint2 every = make_uint2(~0u, ~0u);
  auto load_step = [&](int t, int stage, uint2 shown) {
    const int h = MODE == D_DKV ? oh * group + t / per_head : oh;
    const int at = first + (MODE == D_DKV ? t % per_head : t) * kPart;
    if (MODE == D_DKV) {
      load_rows<T, D>(s_part_a + stage * TILE, q_of(h), p.q_rows.token, at, len.nq, every);
      load_rows<T, D>(s_part_b + stage * TILE, go_of(h), p.go_rows.token, at, len.nq, every);
      if (tid < 64) {
        const int i = at + tid;
        part_lse[stage * 64 + tid] = i < len.nq ? p.lse[stat(h) + i] : INFINITY;
        part_delta[stage * 64 + tid] = i < len.nq ? p.delta[stat(h) + i] : 0.f;
      }
    } else {
      load_rows<T, D>(s_part_a + stage * TILE, K, p.k_rows.token, at, len.nk, shown);
      load_rows<T, D>(s_part_b + stage * TILE, V, p.v_rows.token, at, len.nk, shown);
    }
    if (KIND == MF_BUCKETS_PAIR) load_pairs(MODE == D_DKV ? at : row0, MODE == D_DKV ? row0 : at, stage);
    if (KIND == MF_BUCKETS_OFFSET && tid < kSpan) {  // offsets of the two tiles: owner - partner or partner - owner runs over 127 values
      const int offset = (MODE == D_DKV ? row0 - at + tid - (kPart - 1) : at - row0 + tid - (kOwn - 1)) - len.shift;
      const int bucket = dense_offset_bucket(p, offset);
      offset_bias[stage * 128 + tid] = dense_bias_entry(p, bucket, h);
      if (MODE == D_DQ) offset_bucket[stage * 128 + tid] = (uint8_t)bucket;
    }
  };

  uint2 seen = every, seen_next = every;  // the mask of this tile's keys and of the next one's
  uchar2 bytes = make_uchar2(1, 1);       // of the one after that
  const bool masked = MODE != D_DKV && mask;
  if (steps > 0) {
    if (masked) {
      seen_next = mask_bits(mask_bytes(first));
      bytes = mask_bytes(first + kPart);
    }
    if (MODE == D_DKV) {
      const uint2 shown = mask ? mask_bits(mask_bytes(row0)) : every;
      load_rows<T, D>(s_own_a, K, p.k_rows.token, row0, len.nk, shown);
      load_rows<T, D>(s_own_b, V, p.v_rows.token, row0, len.nk, shown);
    } else {
      load_rows<T, D>(s_own_a, q_of(oh), p.q_rows.token, row0, len.nq, every);
      if (MODE == D_DQ) load_rows<T, D>(s_own_b, go_of(oh), p.go_rows.token, row0, len.nq, every);
    }
    load_step(0, 0, seen_next);
  }
  cp_async_commit();
  if (KIND == MF_BUCKETS_PAIR && MODE == D_FWD)
    for (int i = tid; i < kTableEntries; i += kThreads) table[i] = dense_bias_entry(p, i, oh);

  // ---- visible partners of this thread's two rows: [lo, hi).  Rows that are none see what they want, their results are not used: queries behind the
  // last have a log-sum-exp of infinity, as have partners, so that their p is zero.
  int lo[2], hi[2];
  bool real[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = my + 8 * e;
    real[e] = row < own_limit && (MODE != D_DKV || !mask || mask[row]);
    lo[e] = MODE == D_DKV && real[e] ? dense_first(p, len, row) : 0;
    hi[e] = MODE != D_DKV && real[e] ? dense_limit(p, len, row) : INT32_MAX;
  }
  const int most_lo = __reduce_max_sync(0xffffffffu, max(lo[0], lo[1])), least_hi = __reduce_min_sync(0xffffffffu, min(hi[0], hi[1]));

  float acc0[D / 8][4], acc1[MODE == D_DKV ? D / 8 : 1][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc0[i][e] = 0.f;
  if constexpr (MODE == D_DKV) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc1[i][e] = 0.f;
  }
  const float sc2 = p.scale * kDenseLog2e;
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, lse[2] = {INFINITY, INFINITY}, delta[2] = {0.f, 0.f};
  bool blind[2] = {false, false};  // DQ: queries that see nothing: they and their gradients may hold anything
  if (MODE == D_DQ) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // the four lanes of a row take a quarter of its channels each
      const int row = my + 8 * e;
      float d = 0.f;
      if (row < len.nq) {
        const T* go = go_of(oh) + row * p.go_rows.token + t4 * (D / 4);
        const T* o = static_cast<const T*>(p.out) + p.out_rows.at(b, oh, row) + t4 * (D / 4);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(go + 8 * c), y = *reinterpret_cast<const uint4*>(o + 8 * c);
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = unpack2<T>(xw[i]), w = unpack2<T>(yw[i]);
            d = fmaf(u.x, w.x, fmaf(u.y, w.y, d));
          }
        }
        lse[e] = p.lse[stat(oh) + row];
        blind[e] = lse[e] == INFINITY;
      }
      d += __shfl_xor_sync(0xffffffffu, d, 1);
      d += __shfl_xor_sync(0xffffffffu, d, 2);
      delta[e] = blind[e] ? 0.f : d;
      if (blind[e]) real[e] = false;
    }
  }
  const bool some_blind = MODE == D_DQ && __any_sync(0xffffffffu, blind[0] || blind[1]);
  float error[2] = {0.f, 0.f};  // sums of dS, zero but for what delta is off by


  const bool idle = row0 + warp * 16 >= own_limit;  // a warp without a row brings tiles along and no more
  for (int t = 0; t < steps; ++t) {
    const int stage = STAGES == 2 ? t & 1 : 0;
    const int h = MODE == D_DKV ? oh * group + t / per_head : oh;
    const int at = first + (MODE == D_DKV ? t % per_head : t) * kPart;
    if (masked) {
      seen = seen_next;
      seen_next = mask_bits(bytes);
      bytes = mask_bytes(at + 2 * kPart);
    }
    if (KIND == MF_BUCKETS_PAIR && MODE == D_DKV && t % per_head == 0) {  // another head: another column of the table
      __syncthreads();
      for (int i = tid; i < kTableEntries; i += kThreads) table[i] = dense_bias_entry(p, i, h);
    }
    cp_async_wait<0>();
    __syncthreads();  // tile t has arrived, and everybody is done with the buffers of tile t - 1
    if (STAGES == 2) {
      if (t + 1 < steps) load_step(t + 1, stage ^ 1, seen_next);
      cp_async_commit();
    }
    if constexpr (MODE == D_DKV) {  // queries that see nothing, and their gradients, may hold anything; all warps see the same of them
      auto blind_rows = [&](int i) { return __ballot_sync(0xffffffffu, at + i < len.nq && part_lse[stage * 64 + i] == INFINITY); };
      const uint2 rows = make_uint2(blind_rows(lane), blind_rows(lane + 32));
      if (rows.x | rows.y) {
        uint8_t* tile_at = smem + ((MODE == D_FWD ? 1 : 2) + stage) * TILE;  // part_a; part_b lies STAGES tiles behind it
        for (int idx = tid; idx < 64 * (D / 8); idx += kThreads) {
          const int r = idx / (D / 8), c = idx % (D / 8);
          if (((r & 32 ? rows.y : rows.x) >> (r & 31)) & 1u)
            *reinterpret_cast<uint4*>(tile_at + (r * LD + c * 8) * 2) = *reinterpret_cast<uint4*>(tile_at + STAGES * TILE + (r * LD + c * 8) * 2) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
      }
    }

    if (!idle) {
      const uint32_t pa = s_part_a + stage * TILE, pb = s_part_b + stage * TILE;
      float s[8][4], dp[MODE == D_FWD ? 1 : 8][4];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] = 0.f;
          if constexpr (MODE != D_FWD) dp[nt][e] = 0.f;
        }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4], a2[4];
        ldmatrix_x4(a, s_own_a + ((warp * 16 + (lane & 15)) * LD + ks * 16 + (lane >> 4) * 8) * 2);
        if (MODE != D_FWD) ldmatrix_x4(a2, s_own_b + ((warp * 16 + (lane & 15)) * LD + ks * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
        for (int np = 0; np < 4; ++np) {
          const uint32_t off = ((np * 16 + (lane & 7) + (lane >> 4) * 8) * LD + ks * 16 + ((lane >> 3) & 1) * 8) * 2;
          uint32_t w[4];
          ldmatrix_x4(w, pa + off);
          mma16816<T>(s[2 * np], a, w[0], w[1]);
          mma16816<T>(s[2 * np + 1], a, w[2], w[3]);
          if constexpr (MODE != D_FWD) {
            ldmatrix_x4(w, pb + off);
            mma16816<T>(dp[2 * np], a2, w[0], w[1]);
            mma16816<T>(dp[2 * np + 1], a2, w[2], w[3]);
          }
        }
      }

      // ---- logits in units of log2, minus infinity where nothing is seen
      uint32_t which[KIND == MF_BUCKETS_NONE ? 1 : 8];  // buckets of the 32 elements, a byte each
      if (KIND == MF_BUCKETS_PAIR) {
        const uint8_t* tile_at = pair_tile + stage * kPairTile;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const int c = nt * 8 + 2 * t4, r = warp * 16 + g;
          if (MODE == D_DKV)
            which[nt] = tile_at[c * kPairRow + r] | tile_at[(c + 1) * kPairRow + r] << 8 | tile_at[c * kPairRow + r + 8] << 16 | (uint32_t)tile_at[(c + 1) * kPairRow + r + 8] << 24;
          else
            which[nt] = *reinterpret_cast<const uint16_t*>(tile_at + r * kPairRow + c) | (uint32_t)*reinterpret_cast<const uint16_t*>(tile_at + (r + 8) * kPairRow + c) << 16;
        }
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = nt * 8 + 2 * t4 + (e & 1), r = warp * 16 + g + 8 * (e >> 1);
          if (KIND == MF_BUCKETS_NONE) s[nt][e] *= sc2;
          if (KIND == MF_BUCKETS_OFFSET) s[nt][e] = fmaf(s[nt][e], sc2, offset_bias[stage * 128 + (MODE == D_DKV ? r - c + kPart - 1 : c - r + kOwn - 1)]);
          if (KIND == MF_BUCKETS_PAIR) s[nt][e] = fmaf(s[nt][e], sc2, table[(which[nt] >> (8 * e)) & 255u]);
        }
      if (at < most_lo || at + kPart > least_hi || masked) {
        uint32_t vis[2][2];  // of a row, half of the tile: from the thread's first column on
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          vis[e][0] = (bits_between(lo[e] - at, hi[e] - at) & seen.x) >> (2 * t4);
          vis[e][1] = (bits_between(lo[e] - at - 32, hi[e] - at - 32) & seen.y) >> (2 * t4);
        }
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(vis[e >> 1][nt >> 2] & (1u << ((nt & 3) * 8 + (e & 1))))) s[nt][e] = -INFINITY;
      }

      if (MODE == D_FWD) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = top[e];
#pragma unroll
          for (int nt = 0; nt < 8; ++nt) m = fmaxf(m, fmaxf(s[nt][2 * e], s[nt][2 * e + 1]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float shift = m == -INFINITY ? 0.f : m;
          alpha[e] = dense_exp2(top[e] - shift);
          top[e] = m;
          float sum = 0.f;
#pragma unroll
          for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              s[nt][2 * e + x] = dense_exp2(s[nt][2 * e + x] - shift);
              sum += s[nt][2 * e + x];
            }
          total[e] = total[e] * alpha[e] + sum;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc0[i][e] *= alpha[e >> 1];
      } else {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = nt * 8 + 2 * t4 + (e & 1);
            const float z = s[nt][e];
            const float l = MODE == D_DQ ? lse[e >> 1] : part_lse[stage * 64 + c];
            const float d = MODE == D_DQ ? delta[e >> 1] : part_delta[stage * 64 + c];
            const float pr = dense_exp2(z - l);
            s[nt][e] = pr;
            dp[nt][e] = pr * (dp[nt][e] - d);
            if (MODE == D_DQ) error[e >> 1] += dp[nt][e];
          }
        if (MODE == D_DQ && some_blind) {
#pragma unroll
          for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (blind[e >> 1]) s[nt][e] = dp[nt][e] = 0.f;
          if (blind[0]) error[0] = 0.f;
          if (blind[1]) error[1] = 0.f;
        }
        if (MODE == D_DQ && steps == 1) {  // the whole row is here: its exact delta
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = error[e];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
#pragma unroll
              for (int i = 0; i < 2; ++i) dp[nt][2 * e + i] = fmaf(-x, s[nt][2 * e + i], dp[nt][2 * e + i]);
          }
        }
        if (KIND != MF_BUCKETS_NONE && MODE == D_DQ && p.dbias_part) {
          // a column of sums for every lane: no two threads meet in one, and the order of a sum is that of the walk
#pragma unroll
          for (int nt = 0; nt < 8; ++nt) {
            int bucket[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = nt * 8 + 2 * t4 + (e & 1), r = warp * 16 + g + 8 * (e >> 1);
              bucket[e] = min((int)(KIND == MF_BUCKETS_OFFSET ? offset_bucket[stage * 128 + c - r + kOwn - 1] : (which[nt] >> (8 * e)) & 255u), nb);
            }
            add_four(my_sums, bucket, dp[nt]);
          }
        }
      }

      // ---- products with the partners' rows
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[4], a2[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int nt = 2 * kk + (x >> 1), e = 2 * (x & 1);
          a[x] = pack2<T>(s[nt][e], s[nt][e + 1]);
          if constexpr (MODE != D_FWD) a2[x] = pack2<T>(dp[nt][e], dp[nt][e + 1]);
        }
#pragma unroll
        for (int np = 0; np < D / 16; ++np) {
          const uint32_t off = ((kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * LD + np * 16 + (lane >> 4) * 8) * 2;
          uint32_t w[4];
          if constexpr (MODE == D_FWD) {
            ldmatrix_x4_trans(w, pb + off);
            mma16816<T>(acc0[2 * np], a, w[0], w[1]);
            mma16816<T>(acc0[2 * np + 1], a, w[2], w[3]);
          } else {
            ldmatrix_x4_trans(w, pa + off);
            mma16816<T>(acc0[2 * np], a2, w[0], w[1]);
            mma16816<T>(acc0[2 * np + 1], a2, w[2], w[3]);
          }
          if constexpr (MODE == D_DKV) {
            ldmatrix_x4_trans(w, pb + off);
            mma16816<T>(acc1[2 * np], a, w[0], w[1]);
            mma16816<T>(acc1[2 * np + 1], a, w[2], w[3]);
          }
        }
      }
    }
    if (STAGES == 1) {
      __syncthreads();  // everybody is done with the one buffer
      if (t + 1 < steps) load_step(t + 1, 0, seen_next);
      cp_async_commit();
    }
  }
  cp_async_wait<0>();
  if (MODE == D_DQ) {  // what DKV gets of delta has no rounding of the output in it
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = error[e];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (t4 == 0 && my + 8 * e < p.M) p.delta[stat(oh) + my + 8 * e] = delta[e] + x;
    }
  }

  // ---- rows out: zeros behind the lengths
  float mul[2] = {1.f, 1.f};
  if (MODE == D_FWD) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = total[e];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const bool some = real[e] && (l > 0.f || l != l);
      mul[e] = some ? 1.f / l : 0.f;
      const int row = my + 8 * e;
      if (p.lse && t4 == 0 && row < p.M) p.lse[stat(oh) + row] = some ? top[e] + log2f(l) : INFINITY;
    }
  }
  const int limit = MODE == D_DKV ? p.N : p.M;
  auto store = [&](void* base, const DenseRows& rows, const float (&acc)[D / 8][4], float m0, float m1) {  // a factor of zero: zeros, whatever was summed
    T* dst = static_cast<T*>(base) + rows.at(b, oh, 0);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = my + 8 * e;
      if (row >= limit) continue;
      const float m = e ? m1 : m0;
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt)
        *reinterpret_cast<uint32_t*>(dst + row * rows.token + nt * 8 + 2 * t4) = m == 0.f ? 0u : pack2<T>(acc[nt][2 * e] * m, acc[nt][2 * e + 1] * m);
    }
  };
  if (MODE == D_FWD) store(p.out, p.out_rows, acc0, mul[0], mul[1]);
  const float real0 = real[0] ? 1.f : 0.f, real1 = real[1] ? 1.f : 0.f;
  if (MODE == D_DQ && p.dq) store(p.dq, p.dq_rows, acc0, real0 * p.scale, real1 * p.scale);
  if constexpr (MODE == D_DKV) {
    if (p.dk) store(p.dk, p.dk_rows, acc0, real0 * p.scale, real1 * p.scale);
    if (p.dv) store(p.dv, p.dv_rows, acc1, real0, real1);
  }
  if (STAY) __syncthreads();  // before the next tile's rows arrive
  }
  if (STAY && p.dbias_part) {
    float* part = p.dbias_part + ((long long)(blockIdx.x / heads) * heads + blockIdx.x % heads) * nb;
    for (int i = warp; i < nb; i += 4) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) v += sums[(w * (nb + 1) + i) * 32 + lane];
      v = warp_sum(v);
      if (lane == 0) part[i] = v;
    }
  }
}

// CTAs of a head in the pass that sums the table's gradient: as many as fit the chip, at most one for each tile.
int slots_of(const DenseParams& p, int head_dim) {
  const long long tiles = (long long)p.B * ((p.M + kOwn - 1) / kOwn);
  const int fixed = head_dim == 32   ? Layout<32, D_DQ, MF_BUCKETS_PAIR>::kFixed
                    : head_dim == 64 ? Layout<64, D_DQ, MF_BUCKETS_PAIR>::kFixed
                                     : Layout<128, D_DQ, MF_BUCKETS_PAIR>::kFixed;
  const int smem = fixed + 4 * (p.num_buckets + 1) * 32 * 4 + 1024;
  const int fit = 227 * 1024 / smem, most = 148 * (fit < 1 ? 1 : fit > 3 ? 3 : fit) / p.H;
  return (int)(tiles < most ? tiles : most < 1 ? 1 : most);
}

template <typename T, int D, int MODE, int KIND>
int launch(const DenseParams& p, cudaStream_t stream) {
  const int own = MODE == D_DKV ? p.N : p.M, heads = MODE == D_DKV ? p.K : p.H;
  if (own == 0) return MF_OK;
  const int smem = Layout<D, MODE, KIND>::kFixed + (MODE == D_DQ && KIND != MF_BUCKETS_NONE && p.dbias_part ? 4 * (p.num_buckets + 1) * 32 * 4 : 0);
  constexpr auto kernel = dense_attn_mma_kernel<T, D, MODE, KIND>;
  // one limit for all calls: what the largest table needs
  constexpr int most = Layout<D, MODE, KIND>::kFixed + (MODE == D_DQ && KIND != MF_BUCKETS_NONE ? 4 * (kMaxBuckets + 1) * 32 * 4 : 0);
  static_assert(most <= 227 * 1024, "");
  const cudaError_t err = allow_shared<dense_attn_mma_kernel<T, D, MODE, KIND>>(most);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  const bool stays = MODE == D_DQ && KIND != MF_BUCKETS_NONE && p.dbias_part;
  kernel<<<stays ? slots_of(p, D) * heads : (own + kOwn - 1) / kOwn * p.B * heads, kThreads, smem, stream>>>(p);
  MF_CHECK_LAUNCH("dense attention");
  return MF_OK;
}

template <typename T, int MODE>
int pick(const DenseParams& p, int head_dim, int kind, cudaStream_t stream) {
  auto by_kind = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return kind == MF_BUCKETS_NONE     ? launch<T, D, MODE, MF_BUCKETS_NONE>(p, stream)
           : kind == MF_BUCKETS_OFFSET ? launch<T, D, MODE, MF_BUCKETS_OFFSET>(p, stream)
                                       : launch<T, D, MODE, MF_BUCKETS_PAIR>(p, stream);
  };
  return head_dim == 32   ? by_kind(std::integral_constant<int, 32>{})
         : head_dim == 64 ? by_kind(std::integral_constant<int, 64>{})
                          : by_kind(std::integral_constant<int, 128>{});
}

}  // namespace

int dense_attn_mma_slots(const DenseParams& p, int head_dim) { return p.M ? slots_of(p, head_dim) : 0; }
int dense_attn_mma_fwd(const DenseParams& p, int dtype, int head_dim, int kind, cudaStream_t stream) {
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, D_FWD>(p, head_dim, kind, stream) : pick<__half, D_FWD>(p, head_dim, kind, stream);
}
int dense_attn_mma_bwd(const DenseParams& p, int dtype, int head_dim, int kind, cudaStream_t stream) {
  const int rc = dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, D_DQ>(p, head_dim, kind, stream) : pick<__half, D_DQ>(p, head_dim, kind, stream);
  if (rc != MF_OK || (!p.dk && !p.dv)) return rc;
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, D_DKV>(p, head_dim, kind, stream) : pick<__half, D_DKV>(p, head_dim, kind, stream);
}

}  // namespace mf
