// Dense attention with a learned bias by buckets on tcgen05, forward: head size 64 and 128, bf16 and fp16.
//
// A CTA owns two tiles of 128 query rows (of two heads that share a key head, or neighbours of one head) and walks over the keys in tiles
// of 128, which arrive by bulk tensor copies (boxes of 64 channels, 128-byte swizzle) and serve both.  S = Q K^T lies in tensor memory; a thread owns a
// row of it: it takes the row to registers, and packs P to 16 bits over the first half of the columns that S had, from where it is
// the A operand of O += P V.  While one tile's group of four warps is at its softmax, the tensor cores work for the other: at head size 128 the two
// products of a tile take 1 024 clocks and its exponentials 1 024 (16 a clock), at head size 64 the exponentials bound it.  The accumulator stays
// in tensor memory and is scaled only where a row's maximum has grown by more than 2^8 since it last was; until then P may exceed 1, which
// costs neither type precision.  Sums are of P before it is rounded.  Two tiles of queries in turn and a maximum that is let lag are published methods for
// attention on this generation of tensor cores.  A row's 128 logits in registers leave none over: 4 to 20 bytes a thread are spilled at head size 64, 28 (no bias), 52
// (offset) and 88 (pairs) at 128.
// Two cells of 4096 tokens, 8 heads of 64, with the bias: 122 us, 563 TFLOP/s, exponential unit 61 %; a causal prompt of 4111 fp16 tokens, 16 heads on 4 of 128: 85 us,
// 813 TFLOP/s, exponentials and tensor pipe 46 % each.
//
// Roles: warps 0-3 and 4-7 own the rows of the two tiles, one thread of warp 8 issues the products, one of warp 9 the copies, warp 10 clears the rows
// of V that are no keys (behind the entry's length, or masked), which may hold anything and meet P = 0.  Every wait is bounded; an expired one
// leaves a status word and undefined outputs.
#include "dense_attn_sm100.cuh"

namespace mf {

namespace {

__device__ int32_t g_dense_status[2];  // last expired wait: of calls, of the self-test
__device__ int32_t g_taken_status;
__global__ void take_status_kernel(int word) { g_taken_status = atomicExch(&g_dense_status[word], 0); }

constexpr int kFwdThreads = 384;
// registers: every thread starts with 168; the last four warps drop to kRegAux and the row owners take what that frees
constexpr int kRegAux = 56, kRegOwner = 224;
static_assert(8 * kRegOwner + 4 * kRegAux <= 12 * 168, "register hand-over exceeds the CTA's pool");

template <int D>
struct FwdShape {
  static constexpr int kChunks = D / 64, kTile = kChunks * kTcRows * 128;  // bytes of 128 rows
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kOffQ = 0, kOffRing = 2 * kTile, kSmem = kOffRing + kSlots * kTile + 1024;
  static constexpr int kColO = 256;
};

template <typename T, int D, int KIND>
__global__ void __launch_bounds__(kFwdThreads, 1) dense_attn_tc_kernel(const __grid_constant__ DenseTcParams tc) {
  using Sh = FwdShape<D>;
  const DenseParams& p = tc.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bar_q, bar_full[Sh::kSlots], bar_free[Sh::kSlots], bar_clean[Sh::kSlots], bar_s[2], bar_p[2], bar_o[2], bar_drain;
  __shared__ uint32_t tmem_base;
  __shared__ float table[KIND == MF_BUCKETS_NONE ? 1 : 2][KIND == MF_BUCKETS_NONE ? 1 : kTableEntries];
  __shared__ float offsets[KIND == MF_BUCKETS_OFFSET ? 2 : 1][2][KIND == MF_BUCKETS_OFFSET ? 256 : 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- which rows: two heads of a group, or two neighbouring tiles of a head
  const int group = p.H / p.K;
  const bool by_head = group % 2 == 0;
  const int piece = blockIdx.x % tc.pieces, block = blockIdx.x / tc.pieces, tile0 = piece * tc.piece_tiles;  // of the keys
  const int units = p.B * (by_head ? p.H / 2 : p.H), row_blocks = gridDim.x / tc.pieces / units;
  const int unit = p.causal ? block % units : block / row_blocks;
  const int rb = p.causal ? row_blocks - 1 - block / units : block % row_blocks;  // the longest walks first
  const int b = unit / (units / p.B), hu = unit % (units / p.B);
  const int head0 = by_head ? 2 * hu : hu, kh = head0 / group;
  const DenseLengths len = dense_lengths(p, b);
  int head[2], row0[2], tiles[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    head[x] = by_head ? head0 + x : head0;
    row0[x] = by_head ? rb * kTcRows : (2 * rb + x) * kTcRows;
    const int limit = row0[x] < len.nq ? dense_limit(p, len, min(row0[x] + kTcRows, len.nq) - 1) : 0;
    tiles[x] = max(0, min((limit + kTcRows - 1) / kTcRows - tile0, tc.piece_tiles));
  }
  const int steps = max(tiles[0], tiles[1]);
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.key_mask_batch : nullptr;
  const bool cleaning = mask || len.nk < min(p.N, (tile0 + steps) * kTcRows);

  auto row_out = [&](int x, int r) { return static_cast<T*>(p.out) + p.out_rows.at(b, head[x], row0[x] + r); };
  auto row_stat = [&](int x, int r) -> float& { return p.lse[((long long)b * p.H + head[x]) * p.M + row0[x] + r]; };
  // pieces: where a row leaves its own (see dense_attn_join)
  auto piece_slot = [&](int h, int i) {
    const int row = i * group + h - kh * group, row_tiles = (p.M * group + 15) / 16;
    return (((long long)(b * p.K + kh) * row_tiles + row / 16) * tc.pieces + piece) * 16 + row % 16;
  };
  if (steps == 0) {  // padding only, or nothing is seen
    if (tid < 256) {
      const int x = tid >> 7, r = tid & 127;
      if (row0[x] + r < p.M && tc.pieces > 1) {
        const long long at = piece_slot(head[x], row0[x] + r);
        tc.stat[2 * at] = -INFINITY, tc.stat[2 * at + 1] = 0.f;
      } else if (row0[x] + r < p.M) {
        uint4* dst = reinterpret_cast<uint4*>(row_out(x, r));
        for (int i = 0; i < D / 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
        if (p.lse) row_stat(x, r) = INFINITY;
      }
    }
    return;
  }

  if (tid == 0) {
    auto init = [&](uint64_t* bar, int count, int kind) { mbar_init(bar, count + (tc.waits.withheld == kind)); };
    init(&bar_q, 1, 0);
    for (int i = 0; i < Sh::kSlots; ++i) init(&bar_full[i], 1, 0), init(&bar_free[i], 1, 1), init(&bar_clean[i], 1, 4);
    for (int x = 0; x < 2; ++x) init(&bar_s[x], 1, 2), init(&bar_p[x], 4, 3), init(&bar_o[x], 1, 2);
    mbar_init(&bar_drain, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base;
  const uint32_t s_q = smem_u32(smem + Sh::kOffQ), s_ring = smem_u32(smem + Sh::kOffRing);
  bool bad = false;
  auto wait_on = [&](uint64_t* bar, uint32_t phase) {
    if (!bad) bad = !mbar_wait_for(bar, phase & 1, tc.waits.limit);
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegAux));
  if (warp == 9) {
    // ------------------------------------------------------------------ copies: K of tile j in slot 2 j, V in slot 2 j + 1 (modulo the ring)
    if (lane == 0) {
      tma_prefetch_map(&tc.q);
      tma_prefetch_map(&tc.k);
      tma_prefetch_map(&tc.v);
      const int own = (tiles[0] > 0) + (tiles[1] > 0);
      mbar_arrive_expect_tx(&bar_q, own * Sh::kTile);
      for (int x = 0; x < 2; ++x)
        if (tiles[x] > 0)
          for (int c = 0; c < Sh::kChunks; ++c) tma_box(s_q + x * Sh::kTile + c * kTcRows * 128, &tc.q, c * 64, row0[x], head[x], b, &bar_q);
      int i = 0;
      for (; i < 2 * steps; ++i) {
        const int slot = i % Sh::kSlots;
        if (i >= Sh::kSlots) wait_on(&bar_free[slot], i / Sh::kSlots - 1);
        if (bad) break;
        mbar_arrive_expect_tx(&bar_full[slot], Sh::kTile);
        for (int c = 0; c < Sh::kChunks; ++c)
          tma_box(s_ring + slot * Sh::kTile + c * kTcRows * 128, i & 1 ? &tc.v : &tc.k, c * 64, (tile0 + (i >> 1)) * kTcRows, kh, b, &bar_full[slot]);
      }
      // whoever gave up, no copy may be in flight when the CTA ends
      if (!mbar_wait_for(&bar_q, 0, tc.waits.limit)) bad = true;
      for (int t = max(0, i - Sh::kSlots); t < i; ++t)
        if (!mbar_wait_for(&bar_full[t % Sh::kSlots], (t / Sh::kSlots) & 1, tc.waits.limit)) bad = true;
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ products
    if (elect_one()) {
      const uint32_t l_q = make_desc_lo(s_q, 0), l_k = make_desc_lo(s_ring, 0), l_v = make_desc_lo(s_ring, kTcRows * 128);
      constexpr uint32_t kSlot = Sh::kTile >> 4, kChunk = (kTcRows * 128) >> 4;
      constexpr uint32_t idesc_s = make_idesc_16<T>(kTcRows, kTcRows, false, false), idesc_o = make_idesc_16<T>(kTcRows, D, false, true);
      auto logits = [&](int x, int slot) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * kChunk + (ks & 3) * 2;
          umma_ss_lo(tmem + 128 * x, l_q + x * kSlot + off, l_k + slot * kSlot + off, idesc_s, ks > 0);
        }
        umma_commit(&bar_s[x]);
      };
      wait_on(&bar_q, 0);
      wait_on(&bar_full[0], 0);
      tc_fence_after_sync();
      for (int x = 0; x < 2; ++x)
        if (tiles[x] > 0) logits(x, 0);
      umma_commit(&bar_free[0]);
      for (int j = 0; j < steps; ++j) {
        const int iv = 2 * j + 1, vs = iv % Sh::kSlots, ik = iv + 1, ks_ = ik % Sh::kSlots;
        wait_on(cleaning ? &bar_clean[vs] : &bar_full[vs], iv / Sh::kSlots);
        if (j + 1 < steps) wait_on(&bar_full[ks_], ik / Sh::kSlots);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (j >= tiles[x]) continue;
          wait_on(&bar_p[x], j);
          tc_fence_after_sync();
#pragma unroll
          for (int kg = 0; kg < kTcRows / 16; ++kg)
            umma_ts_lo(tmem + Sh::kColO + D * x, tmem + 128 * x + 8 * kg, l_v + vs * kSlot + 128 * kg, idesc_o, j > 0 || kg > 0);
          if (j + 1 < tiles[x]) logits(x, ks_);
          else umma_commit(&bar_o[x]);
        }
        umma_commit(&bar_free[vs]);
        if (j + 1 < steps) umma_commit(&bar_free[ks_]);
      }
      // nor a product when tensor memory is given back
      umma_commit(&bar_drain);
      if (!mbar_wait(&bar_drain, 0)) bad = true;
    }
  } else if (warp == 10) {
    // ------------------------------------------------------------------ rows of V that are no keys become zeros
    if (cleaning) {
      for (int j = 0; j < steps; ++j) {
        const int iv = 2 * j + 1, slot = iv % Sh::kSlots;
        wait_on(&bar_full[slot], iv / Sh::kSlots);
        const int first = (tile0 + j) * kTcRows, last = min(kTcRows, p.N - first);  // rows behind the tensor's are zeros already
        if (!bad && (mask || first + last > len.nk)) {
          for (int r = lane; r < last; r += 32) {
            const int key = first + r;
            if (key < len.nk && (!mask || mask[key])) continue;
#pragma unroll
            for (int c = 0; c < Sh::kChunks; ++c)
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(smem + Sh::kOffRing + slot * Sh::kTile + c * kTcRows * 128 + r * 128 + i * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_smem_to_async_proxy();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_clean[slot]);
      }
    }
  }
  } else {
    // ------------------------------------------------------------------ row owners
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegOwner));
    const int x = warp >> 2, r = tid & 127;
    const int my_head = x ? head[1] : head[0], my_row0 = x ? row0[1] : row0[0], my_tiles = x ? tiles[1] : tiles[0];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t col_s = tmem + lanes + 128 * x, col_o = tmem + lanes + Sh::kColO + D * x;
    const int i = my_row0 + r;
    const bool row_ok = i < len.nq;
    // a row that is no query may see what it wants: its result is not used
    const int limit = row_ok ? dense_limit(p, len, i) : INT32_MAX;
    const int least = __reduce_min_sync(0xffffffffu, limit);
    const float sc2 = p.scale * kDenseLog2e;
    float top = -INFINITY, total = 0.f;
    float far[2] = {0.f, 0.f};  // bias of the offsets -reach and reach, and beyond
    if (KIND != MF_BUCKETS_NONE) {
      for (int e = r; e < kTableEntries; e += 128) table[x][e] = dense_bias_entry(p, e, my_head);
      group_barrier(1 + x, 128);
      if (KIND == MF_BUCKETS_OFFSET) far[0] = table[x][p.buckets[0]], far[1] = table[x][p.buckets[2 * p.reach]];
    }
    const uint8_t* pair_row = KIND == MF_BUCKETS_PAIR ? p.buckets + b * p.bucket_batch + min(i, p.M - 1) * p.bucket_row : nullptr;
    int fills = 0;
    for (int j = 0; j < my_tiles; ++j) {
      const int key0 = (tile0 + j) * kTcRows;
      float one = 0.f;
      const float* near = nullptr;
      if (KIND == MF_BUCKETS_OFFSET) {
        const int start = key0 - my_row0 - len.shift - 127;  // the offset of entry 0; entry e stands for the columns c of rows r with c - r = e - 127
        if (start + 254 <= -p.reach) {
          one = far[0];
        } else if (start >= p.reach) {
          one = far[1];
        } else {
          float* values = offsets[x][fills & 1];
          const int b0 = dense_offset_bucket(p, start + r), b1 = dense_offset_bucket(p, start + r + 128);
          values[r] = table[x][b0], values[r + 128] = table[x][b1];
          group_barrier(1 + x, 128);
          near = values + 127 - r;
          ++fills;
        }
      }
      uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
      if (mask) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int key = key0 + 32 * w + lane;
          seen[w] = __ballot_sync(0xffffffffu, key < len.nk && mask[key] != 0);
        }
      }
      wait_on(&bar_s[x], j);
      tc_fence_after_sync();
      float z[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(col_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&z[32 * c]));
      tmem_ld_wait();
      if (KIND == MF_BUCKETS_OFFSET && near) {
#pragma unroll
        for (int c = 0; c < 128; ++c) z[c] = fmaf(z[c], sc2, near[c]);
      } else if (KIND == MF_BUCKETS_PAIR) {
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          uint32_t w[4] = {0, 0, 0, 0};
          if (key0 + c + 16 <= p.N) {
            const uint4 v = *reinterpret_cast<const uint4*>(pair_row + key0 + c);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (key0 + c + e < p.N) w[e >> 2] |= (uint32_t)pair_row[key0 + c + e] << (8 * (e & 3));
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) z[c + e] = fmaf(z[c + e], sc2, table[x][(w[e >> 2] >> (8 * (e & 3))) & 255u]);
        }
      }
      // z is the logit where pairs have biases of their own; otherwise z * mul + one is, and its maximum is formed from z's
      const bool own_bias = KIND == MF_BUCKETS_PAIR || (KIND == MF_BUCKETS_OFFSET && near);
      float mul = own_bias ? 1.f : sc2;
      if (mul <= 0.f) {  // (a maximum of products is not the product of the maximum)
#pragma unroll
        for (int c = 0; c < 128; ++c) z[c] *= mul;
        mul = 1.f;
      }
      if (key0 + kTcRows > least || mask) {
        const int left = limit - key0;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c >= left || !((seen[c >> 5] >> (c & 31)) & 1u)) z[c] = -INFINITY;
      }
      float m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        m[q] = z[32 * q];
#pragma unroll
        for (int c = 1; c < 31; c += 2) m[q] = max3(m[q], z[32 * q + c], z[32 * q + c + 1]);
        m[q] = fmaxf(m[q], z[32 * q + 31]);
      }
      const float mine = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      const float now = fmaxf(top, mine == -INFINITY ? mine : fmaf(mine, mul, one));
      if (j == 0) {
        top = now;
      } else if (__any_sync(0xffffffffu, now > top + 8.f)) {
        const float alpha = now == -INFINITY ? 1.f : dense_exp2(top - now);
        total *= alpha;
        top = now;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(col_o + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st16(col_o + c, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
          tmem_st16(col_o + c + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
        }
      }
      const float shift = one == -INFINITY ? one : top == -INFINITY ? 0.f : one - top;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 v = fma2(make_float2(z[c + e], z[c + e + 1]), make_float2(mul, mul), make_float2(shift, shift));
          v.x = dense_exp2(v.x), v.y = dense_exp2(v.y);
          sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], v);
          w[e >> 1] = pack2<T>(v.x, v.y);
        }
        tmem_st16(col_s + (c >> 1), w);
      }
      total += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[x]);
    }
    if (my_tiles > 0) wait_on(&bar_o[x], 0);
    tc_fence_after_sync();
    const bool some = row_ok && (total > 0.f || total != total);
    const float inv = some ? 1.f / total : 0.f;
    const long long slot = tc.pieces > 1 && i < p.M ? piece_slot(my_head, i) : 0;
#pragma unroll
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      if (my_tiles > 0) {
        tmem_ld32(col_o + c, o);
        tmem_ld_wait();
      }
      if (tc.pieces > 1) {
        if (i < p.M && some)
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(tc.acc + slot * D + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      } else if (i < p.M) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + p.out_rows.at(b, my_head, i) + c);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) w[y] = some ? pack2<T>(__uint_as_float(o[e + 2 * y]) * inv, __uint_as_float(o[e + 2 * y + 1]) * inv) : 0u;
          dst[e >> 3] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (tc.pieces > 1) {
      if (i < p.M) tc.stat[2 * slot] = some ? top : -INFINITY, tc.stat[2 * slot + 1] = some ? total : 0.f;
    } else if (p.lse && i < p.M) {
      p.lse[((long long)b * p.H + my_head) * p.M + i] = some ? top + log2f(total) : INFINITY;
    }
    tc_fence_before_sync();
  }
  if (bad) atomicExch(&g_dense_status[tc.waits.word], MF_ERR_DEVICE_TIMEOUT);
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// CTAs without pieces of the keys.
long long blocks_of(const DenseParams& p) {
  const long long tiles = (p.M + kTcRows - 1) / kTcRows;
  return (p.H / p.K) % 2 == 0 ? tiles * p.B * (p.H / 2) : (tiles + 1) / 2 * p.B * p.H;
}
// Pieces of the keys: where the tiles of the queries would fill less than half of the SMs through long walks, as many as the SMs hold, of four tiles at least.
// (Microseconds with | without: 2611 queries, 2 heads of 128 on one, 6412 keys 31 | 94; 512 queries, 8 heads of 64, 2048 keys 17 | 33, 4096 keys 20 | 61; 4111 causal, 4 heads of
// 128 on one 53 | 70.)
int pieces_of(const DenseParams& p) {
  const long long blocks = blocks_of(p), tiles = (p.N + kTcRows - 1) / kTcRows;
  if (blocks * 2 > 148 || tiles < 16) return 1;
  const long long most = 148 / blocks < tiles / 4 ? 148 / blocks : tiles / 4, size = (tiles + most - 1) / most;
  return (int)((tiles + size - 1) / size);
}

template <typename T, int D, int KIND>
int launch(DenseTcParams& tc, void* workspace, cudaStream_t stream) {
  const DenseParams& p = tc.p;
  const int tiles = (p.N + kTcRows - 1) / kTcRows;
  tc.pieces = pieces_of(p), tc.piece_tiles = (tiles + tc.pieces - 1) / tc.pieces;
  if (tc.pieces > 1) {
    tc.acc = static_cast<float*>(workspace);
    tc.stat = tc.acc + (long long)p.B * p.K * (((long long)p.M * (p.H / p.K) + 15) / 16) * tc.pieces * 16 * D;
  }
  constexpr auto kernel = dense_attn_tc_kernel<T, D, KIND>;
  const cudaError_t err = allow_shared<dense_attn_tc_kernel<T, D, KIND>>(FwdShape<D>::kSmem);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  kernel<<<(unsigned)(blocks_of(p) * tc.pieces), kFwdThreads, FwdShape<D>::kSmem, stream>>>(tc);
  MF_CHECK_LAUNCH("dense attention on tcgen05");
  if (tc.pieces > 1) return dense_attn_join(p, std::is_same<T, __half>::value ? MF_DTYPE_F16 : MF_DTYPE_BF16, D, tc.pieces, tc.acc, tc.stat, stream);
  return MF_OK;
}

template <typename T>
int pick(DenseTcParams& tc, int head_dim, int kind, void* workspace, cudaStream_t stream) {
  auto by_kind = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return kind == MF_BUCKETS_NONE     ? launch<T, D, MF_BUCKETS_NONE>(tc, workspace, stream)
           : kind == MF_BUCKETS_OFFSET ? launch<T, D, MF_BUCKETS_OFFSET>(tc, workspace, stream)
                                       : launch<T, D, MF_BUCKETS_PAIR>(tc, workspace, stream);
  };
  return head_dim == 64 ? by_kind(std::integral_constant<int, 64>{}) : by_kind(std::integral_constant<int, 128>{});
}

bool rows_map(CUtensorMap* map, const void* base, const DenseRows& rows, int dtype, int head_dim, int tokens, int heads, int batch, int box_rows) {
  const long long dims[4] = {head_dim, tokens, heads, batch};
  long long strides[3] = {rows.token * 2, rows.head * 2, rows.batch * 2};
  for (int i = 0; i < 3; ++i)
    if (dims[i + 1] == 1) strides[i] = head_dim * 2;  // whatever it is, nothing goes by it
  for (int i = 0; i < 3; ++i)
    if (strides[i] <= 0) return false;  // (an expanded dimension)
  return make_tensor_map(map, base, dtype, 4, dims, strides, 64, box_rows);
}

}  // namespace

int dense_attn_take_fwd_status(int word, int32_t* host_status, cudaStream_t stream) {
  take_status_kernel<<<1, 1, 0, stream>>>(word);
  MF_CHECK_LAUNCH("dense attention status read-back");
  cudaError_t e = cudaMemcpyFromSymbolAsync(host_status, g_taken_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "dense attention status read-back");
}

bool dense_tc_maps(DenseTcParams& tc, int dtype, int head_dim, bool backward) {
  const DenseParams& p = tc.p;
  const int box = backward ? 64 : kTcRows;
  return rows_map(&tc.q, p.q, p.q_rows, dtype, head_dim, p.M, p.H, p.B, box) && rows_map(&tc.k, p.k, p.k_rows, dtype, head_dim, p.N, p.K, p.B, box) &&
         rows_map(&tc.v, p.v, p.v_rows, dtype, head_dim, p.N, p.K, p.B, box) &&
         (!backward || rows_map(&tc.grad_out, p.grad_out, p.go_rows, dtype, head_dim, p.M, p.H, p.B, box));
}

bool dense_tc_takes(const DenseParams& p, int head_dim, int kind) {
  if (head_dim == 32 || p.M < 1 || p.N < 1) return false;
  if (kind == MF_BUCKETS_PAIR && (reinterpret_cast<uintptr_t>(p.buckets) % 16 || p.bucket_row % 16 || p.bucket_batch % 16)) return false;  // read 16 at a time
  return p.M <= 1 << 24 && p.N <= 1 << 24;
}

size_t dense_tc_fwd_workspace_bytes(const DenseParams& p, int head_dim) {
  const int pieces = pieces_of(p);
  return pieces > 1 ? dense_attn_join_bytes(p, head_dim, pieces) : 0;
}
int dense_attn_sm100_fwd(const DenseParams& p, int dtype, int head_dim, int kind, void* workspace, cudaStream_t stream, BoundedWaits waits) {
  DenseTcParams tc{p, {}, {}, {}, {}, waits};
  if (!dense_tc_maps(tc, dtype, head_dim, false)) return dense_attn_mma_fwd(p, dtype, head_dim, kind, stream);
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16>(tc, head_dim, kind, workspace, stream) : pick<__half>(tc, head_dim, kind, workspace, stream);
}

}  // namespace mf
