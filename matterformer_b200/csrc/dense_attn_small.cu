// Dense attention with a learned bias by buckets on at most 32 queries and 32 keys (small molecules): a warp for every (entry, head), its logits, probabilities
// and their gradients whole in registers.
//
// The operands of an item are 32 rows each in the warp's own part of shared memory (cp.async in, 16-byte rows out, both coalesced); nothing is
// shared between warps, so they drift apart and hide each other's latencies.  A row of the softmax lies in four lanes: its maximum, sum and, backward,
// delta = sum_j p_j dP_j are exact sums of what the warp holds, and `out` is not read again.  P and dS are transposed in 8 x 8 tiles
// (movmatrix) where a product runs over the queries.  The keys are taken in an order in which the eight of a row that a lane holds are neighbours, so that their
// buckets are two words and their visibility a byte.  Warps stay with one head and walk over the entries, so the table's gradient is summed per
// lane in shared memory over the whole walk and leaves once.  An item of 29 tokens and 64 channels is 15 KB forward, 26 KB backward, for 1.7 and 4.3 MFLOP
// with the padding: what bounds it is the latency of an item's chain and the instructions around the
// products (42 to 55 % of the issue slots). 1024 molecules of 9 to 29 tokens, 8 heads of 64: forward 26 us, backward 51 (2.4 TB/s).
#include "dense_attn.cuh"

namespace mf {
namespace {

constexpr int kWarps = 2, kN = 32;

template <int D>
constexpr int kTile = kN * D * 2;

// The key of column c (0 .. 7) of the column tile nt: lane t of a row holds c = 2 t and 2 t + 1 of all four tiles, keys 8 t .. 8 t + 7.
__device__ __forceinline__ int key_of(int nt, int c) { return (c >> 1) * 8 + nt * 2 + (c & 1); }
// Rows of D channels without padding, whose 16-byte chunks change places so that the eight rows that a matrix load takes lie in different banks: rows in
// their order for queries, those of key_of for keys.
template <int D>
__device__ __forceinline__ uint32_t q_place(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (D == 32 ? (row >> 1) & 3 : row & 7)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t k_place(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (D == 32 ? (row >> 3) & 3 : (row & 1) | ((row >> 2) & 6))) << 4);
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// rows [0, n) of a head into the warp's tile, zeros behind them and where `shown` has no bit
template <typename T, int D, bool KEYS>
__device__ __forceinline__ void rows_in(uint32_t tile, const T* src, long long stride, int n, uint32_t shown, int lane) {
  constexpr int CHUNKS = D / 8, ROWS = 32 / CHUNKS;
  const int r0 = lane / CHUNKS, c = lane % CHUNKS;
  const T* at = src + r0 * stride + c * 8;
  const uint32_t ok = (n >= 32 ? 0xffffffffu : (1u << n) - 1u) & shown;
#pragma unroll
  for (int it = 0; it < kN / ROWS; ++it) {
    const int r = it * ROWS + r0;
    const bool there = (ok >> r) & 1u;
    cp_async16(tile + (KEYS ? k_place<D>(r, c) : q_place<D>(r, c)), there ? at : src, there);
    at += ROWS * stride;
  }
}
template <typename T, int D, bool KEYS>
__device__ __forceinline__ void rows_out(T* dst, long long stride, int rows, const uint8_t* tile, int lane) {
  constexpr int CHUNKS = D / 8, ROWS = 32 / CHUNKS;
  const int r0 = lane / CHUNKS, c = lane % CHUNKS;
  T* at = dst + r0 * stride + c * 8;
#pragma unroll
  for (int it = 0; it < kN / ROWS; ++it) {
    const int r = it * ROWS + r0;
    if (r < rows) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(tile + (KEYS ? k_place<D>(r, c) : q_place<D>(r, c)));
    at += ROWS * stride;
  }
}
// a 16 x D accumulator into rows r0 (of lane group g) and r1 of a tile; a factor of zero gives zeros whatever was summed
template <typename T, int D, bool KEYS>
__device__ __forceinline__ void keep(uint8_t* tile, int r0, int r1, const float (&acc)[D / 8][4], float m0, float m1, int lane) {
  const int t4 = lane & 3;
#pragma unroll
  for (int nt = 0; nt < D / 8; ++nt) {
    const uint32_t a = KEYS ? k_place<D>(r0, nt) : q_place<D>(r0, nt), b = KEYS ? k_place<D>(r1, nt) : q_place<D>(r1, nt);
    *reinterpret_cast<uint32_t*>(tile + a + 4 * t4) = m0 == 0.f ? 0u : pack2<T>(acc[nt][0] * m0, acc[nt][1] * m0);
    *reinterpret_cast<uint32_t*>(tile + b + 4 * t4) = m1 == 0.f ? 0u : pack2<T>(acc[nt][2] * m1, acc[nt][3] * m1);
  }
}
// s (16 x 32) = rows [row0, row0 + 16) of a query tile . rows of a key tile, in the order of key_of
template <typename T, int D>
__device__ __forceinline__ void product(float (&s)[4][4], uint32_t a_tile, int row0, uint32_t b_tile, int lane) {
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
  const int key0 = key_of(lane >> 4, lane & 7);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    uint32_t a[4], w[4];
    ldmatrix_x4(a, a_tile + q_place<D>(row0 + (lane & 15), ks * 2 + (lane >> 4)));
#pragma unroll
    for (int np = 0; np < 2; ++np) {
      ldmatrix_x4(w, b_tile + k_place<D>(key0 + 4 * np, ks * 2 + ((lane >> 3) & 1)));
      mma16816<T>(s[2 * np], a, w[0], w[1]);
      mma16816<T>(s[2 * np + 1], a, w[2], w[3]);
    }
  }
}
// acc (16 x D) = a (16 x 32, packed) . rows of a tile: keys in the order of key_of, or queries
template <typename T, int D, bool KEYS>
__device__ __forceinline__ void contract(float (&acc)[D / 8][4], const uint32_t (&a)[2][4], uint32_t b_tile, bool both, int lane) {
#pragma unroll
  for (int nt = 0; nt < D / 8; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    if (kk == 1 && !both) continue;
    const int row = KEYS ? key_of(2 * kk + ((lane >> 3) & 1), lane & 7) : kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
      uint32_t w[4];
      const int chunk = np * 2 + (lane >> 4);
      ldmatrix_x4_trans(w, b_tile + (KEYS ? k_place<D>(row, chunk) : q_place<D>(row, chunk)));
      mma16816<T>(acc[2 * np], a[kk], w[0], w[1]);
      mma16816<T>(acc[2 * np + 1], a[kk], w[2], w[3]);
    }
  }
}

struct SmallParams {
  DenseParams p;
  int slots;  // warps of a head
};

// Shared memory of a warp: tiles of Q K V (dO), the head's column of the table with one entry for buckets beyond it (or the 64 offsets' bias and buckets behind it),
// backward a column of sums for every lane.
template <int D, bool BWD>
constexpr int kTilesBytes = (BWD ? 4 : 3) * kTile<D>;
__host__ __device__ constexpr int small_table_bytes(int kind, int nb) {
  return kind == MF_BUCKETS_NONE ? 0 : (4 * (nb + 1) + (kind == MF_BUCKETS_OFFSET ? 64 * 4 + 64 : 0) + 15) / 16 * 16;
}

template <typename T, int D, int KIND, bool BWD>
__global__ void __launch_bounds__(kWarps * 32, BWD || D == 128 ? 5 : 8) dense_attn_small_kernel(const __grid_constant__ SmallParams sp) {
  const DenseParams& p = sp.p;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int nb = p.num_buckets;
  const bool table_grad = BWD && KIND != MF_BUCKETS_NONE && p.dbias_part;
  uint8_t* mine = smem + warp * kTilesBytes<D, BWD>;
  uint8_t *t_q = mine, *t_k = mine + kTile<D>, *t_v = mine + 2 * kTile<D>, *t_o = mine + 3 * kTile<D>;
  const uint32_t s_q = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), s_k = s_q + kTile<D>, s_v = s_k + kTile<D>, s_o = s_v + kTile<D>;
  const int table_bytes = small_table_bytes(KIND, nb);
  float* table = reinterpret_cast<float*>(smem + kWarps * kTilesBytes<D, BWD> + warp * table_bytes);
  float* offset_bias = table + nb + 1;
  uint8_t* offset_bucket = reinterpret_cast<uint8_t*>(offset_bias + 64);
  float* sums = reinterpret_cast<float*>(smem + kWarps * (kTilesBytes<D, BWD> + table_bytes)) + warp * (nb + 1) * 32 + lane;
  launch_dependents();
  wait_for_previous();

  const int id = blockIdx.x * kWarps + warp, h = id % p.H, slot = id / p.H;
  if (slot >= sp.slots) return;
  const int kh = h / (p.H / p.K);
  if (KIND != MF_BUCKETS_NONE) {
    for (int i = lane; i <= nb; i += 32) table[i] = dense_bias_entry(p, i, h);
    __syncwarp();
  }
  if (table_grad)
    for (int i = 0; i <= nb; ++i) sums[i * 32] = 0.f;
  const float sc2 = p.scale * kDenseLog2e;
  const uint32_t nb4 = (uint32_t)nb * 0x01010101u;

  for (int b = slot; b < p.B; b += sp.slots) {
    const DenseLengths len = dense_lengths(p, b);
    uint32_t shown = 0xffffffffu;
    if (p.key_mask) shown = __ballot_sync(0xffffffffu, lane < p.N && p.key_mask[b * p.key_mask_batch + lane] != 0);
    rows_in<T, D, false>(s_q, static_cast<const T*>(p.q) + p.q_rows.at(b, h, 0), p.q_rows.token, len.nq, 0xffffffffu, lane);
    rows_in<T, D, true>(s_k, static_cast<const T*>(p.k) + p.k_rows.at(b, kh, 0), p.k_rows.token, len.nk, shown, lane);
    rows_in<T, D, true>(s_v, static_cast<const T*>(p.v) + p.v_rows.at(b, kh, 0), p.v_rows.token, len.nk, shown, lane);
    if (BWD) rows_in<T, D, false>(s_o, static_cast<const T*>(p.grad_out) + p.go_rows.at(b, h, 0), p.go_rows.token, len.nq, 0xffffffffu, lane);
    cp_async_commit();
    float* stat = p.lse ? p.lse + ((long long)b * p.H + h) * p.M : nullptr;

    // of the thread's four rows (g, g + 8, g + 16, g + 24): whether it sees its eight keys, a bit each, and their buckets, a byte each
    uint32_t see[4];
    uint2 bucket[KIND == MF_BUCKETS_PAIR ? 4 : 1];
    float lse[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = g + 8 * x, limit = dense_limit(p, len, i);
      see[x] = ((limit >= 32 ? 0xffffffffu : (1u << limit) - 1u) & shown) >> (8 * t4);
      if (BWD) lse[x] = i < len.nq ? stat[i] : INFINITY;
      if (KIND == MF_BUCKETS_PAIR) {
        uint2 w = eight_bytes(p.buckets + b * p.bucket_batch + i * p.bucket_row + 8 * t4, i < len.nq ? p.N - 8 * t4 : 0);
        bucket[x] = make_uint2(__vminu4(w.x, nb4), __vminu4(w.y, nb4));
      }
    }
    if (KIND == MF_BUCKETS_OFFSET) {  // entry e: offset e - 31 from key 0 and query 31 on
#pragma unroll
      for (int e = lane; e < 64; e += 32) {
        const int at = min(dense_offset_bucket(p, e - 31 - len.shift), nb);
        offset_bucket[e] = (uint8_t)at;
        offset_bias[e] = table[at];
      }
    }
    // element k (of eight) of row x
    auto bucket_of = [&](int x, int k) {
      if (KIND == MF_BUCKETS_OFFSET) return (int)offset_bucket[8 * t4 + k - g - 8 * x + 31];
      return (int)(((k < 4 ? bucket[KIND == MF_BUCKETS_PAIR ? x : 0].x : bucket[KIND == MF_BUCKETS_PAIR ? x : 0].y) >> (8 * (k & 3))) & 255u);
    };
    const bool q2 = len.nq > 16;
    cp_async_wait<0>();
    __syncwarp();
    if constexpr (BWD) {  // queries that see nothing, and their gradients, may hold anything
      auto blind = [&](int x) { return g + 8 * x < len.nq && lse[x] == INFINITY; };
      if (__any_sync(0xffffffffu, blind(0) || blind(1) || blind(2) || blind(3))) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          for (int c = t4; blind(x) && c < D / 8; c += 4)
            *reinterpret_cast<uint4*>(t_q + q_place<D>(g + 8 * x, c)) = *reinterpret_cast<uint4*>(t_o + q_place<D>(g + 8 * x, c)) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
    }

    uint32_t P[2][2][4], S[BWD ? 2 : 1][2][4];  // packed, [query half][pair of column tiles]: A operands of products over the keys
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      if (mt == 1 && !q2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          P[1][i >> 2][i & 3] = 0u;
          if constexpr (BWD) S[1][i >> 2][i & 3] = 0u;
        }
        continue;
      }
      float s[4][4], dp[BWD ? 4 : 1][4];
      product<T, D>(s, s_q, mt * 16, s_k, lane);
      if constexpr (BWD) product<T, D>(dp, s_o, mt * 16, s_v, lane);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 2 * mt + x;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float& z = s[k >> 1][2 * x + (k & 1)];
          if (KIND == MF_BUCKETS_NONE) z *= sc2;
          else if (KIND == MF_BUCKETS_OFFSET) z = fmaf(z, sc2, offset_bias[8 * t4 + k - g - 8 * row + 31]);
          else z = fmaf(z, sc2, table[bucket_of(row, k)]);
          z = (see[row] >> k) & 1u ? z : -INFINITY;
          if (!BWD) m = fmaxf(m, z);
        }
        if constexpr (!BWD) {
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float shift = m == -INFINITY ? 0.f : m;
          float l = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float& z = s[k >> 1][2 * x + (k & 1)];
            l += z = dense_exp2(z - shift);
          }
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const int i = g + 8 * row;
          const bool some = l > 0.f || l != l;
          if (stat && t4 == 0 && i < p.M) stat[i] = some ? m + log2f(l) : INFINITY;
          lse[row] = some ? 1.f / l : 0.f;
        } else {
          float d = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float &z = s[k >> 1][2 * x + (k & 1)], &o = dp[k >> 1][2 * x + (k & 1)];
            const float pr = (see[row] >> k) & 1u ? dense_exp2(z - lse[row]) : 0.f;
            z = pr;
            o = pr == 0.f ? 0.f : o;
            d = fmaf(pr, o, d);
          }
          d += __shfl_xor_sync(0xffffffffu, d, 1);
          d += __shfl_xor_sync(0xffffffffu, d, 2);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float& o = dp[k >> 1][2 * x + (k & 1)];
            o = s[k >> 1][2 * x + (k & 1)] * (o - d);
          }
          if (table_grad) {  // a column of sums for every lane: no two threads meet in one
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
              const int at[4] = {bucket_of(row, k), bucket_of(row, k + 1), bucket_of(row, k + 2), bucket_of(row, k + 3)};
              const float d4[4] = {dp[k >> 1][2 * x], dp[k >> 1][2 * x + 1], dp[(k >> 1) + 1][2 * x], dp[(k >> 1) + 1][2 * x + 1]};
              add_four(sums, at, d4);
            }
          }
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int nt = 2 * kk + (x >> 1), e = 2 * (x & 1);
          P[mt][kk][x] = pack2<T>(s[nt][e], s[nt][e + 1]);
          if constexpr (BWD) S[mt][kk][x] = pack2<T>(dp[nt][e], dp[nt][e + 1]);
        }
    }

    float acc[D / 8][4];
    if constexpr (!BWD) {
      __syncwarp();  // the queries have been read: their tile takes the result
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        if (mt == 1 && p.M <= 16) continue;
        contract<T, D, true>(acc, P[mt], s_v, true, lane);
        keep<T, D, false>(t_q, mt * 16 + g, mt * 16 + g + 8, acc, mt && !q2 ? 0.f : lse[2 * mt], mt && !q2 ? 0.f : lse[2 * mt + 1], lane);
      }
      if (!q2 && stat && t4 == 0)
#pragma unroll
        for (int x = 2; x < 4; ++x)
          if (g + 8 * x < p.M) stat[g + 8 * x] = INFINITY;
      __syncwarp();
      rows_out<T, D, false>(static_cast<T*>(p.out) + p.out_rows.at(b, h, 0), p.out_rows.token, p.M, t_q, lane);
    } else {
      __syncwarp();  // the values have been read
      if (p.dq) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          if (mt == 1 && p.M <= 16) continue;
          const int r0 = mt * 16 + g, r1 = r0 + 8;
          contract<T, D, true>(acc, S[mt], s_k, true, lane);
          keep<T, D, false>(t_v, r0, r1, acc, r0 < len.nq ? p.scale : 0.f, r1 < len.nq ? p.scale : 0.f, lane);
        }
        __syncwarp();  // and the keys
        rows_out<T, D, false>(static_cast<T*>(p.dq) + p.dq_rows.at(b, h, 0), p.dq_rows.token, p.M, t_v, lane);
      }
      auto turned = [&](uint32_t (&a)[2][4], const uint32_t (&x)[2][2][4], int kk) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          a[mt][0] = transposed(x[mt][kk][0]), a[mt][1] = transposed(x[mt][kk][2]);
          a[mt][2] = transposed(x[mt][kk][1]), a[mt][3] = transposed(x[mt][kk][3]);
        }
      };
      auto real = [&](int j) { return j < len.nk && ((shown >> j) & 1u); };
      uint32_t a[2][4];
      if (p.dv) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const int r0 = key_of(2 * kk, g), r1 = key_of(2 * kk + 1, g);
          turned(a, P, kk);
          contract<T, D, false>(acc, a, s_o, q2, lane);
          keep<T, D, true>(t_k, r0, r1, acc, real(r0) ? 1.f : 0.f, real(r1) ? 1.f : 0.f, lane);
        }
        __syncwarp();
        rows_out<T, D, true>(static_cast<T*>(p.dv) + p.dv_rows.at(b, kh, 0), p.dv_rows.token, p.N, t_k, lane);
      }
      if (p.dk) {
        __syncwarp();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const int r0 = key_of(2 * kk, g), r1 = key_of(2 * kk + 1, g);
          turned(a, S, kk);
          contract<T, D, false>(acc, a, s_q, q2, lane);
          keep<T, D, true>(t_o, r0, r1, acc, real(r0) ? p.scale : 0.f, real(r1) ? p.scale : 0.f, lane);
        }
        __syncwarp();
        rows_out<T, D, true>(static_cast<T*>(p.dk) + p.dk_rows.at(b, kh, 0), p.dk_rows.token, p.N, t_o, lane);
      }
    }
    __syncwarp();  // before the next entry's rows arrive
  }
  if (table_grad) {
    __syncwarp();
    float* part = p.dbias_part + ((long long)slot * p.H + h) * nb;
    for (int i = 0; i < nb; ++i) {
      const float v = warp_sum(sums[i * 32]);
      if (lane == 0) part[i] = v;
    }
  }
}

int smem_of(const DenseParams& p, int head_dim, int kind, bool bwd, bool table_grad) {
  return kWarps * ((bwd ? 4 : 3) * kN * head_dim * 2 + small_table_bytes(kind, p.num_buckets) + (table_grad ? (p.num_buckets + 1) * 32 * 4 : 0));
}
// Warps of a head: as many as fit the chip, at most one for each entry.
int slots_of(const DenseParams& p, int head_dim, int kind, bool bwd, bool table_grad) {
  const int fit = 227 * 1024 / (smem_of(p, head_dim, kind, bwd, table_grad) + 1024), regs = bwd || head_dim == 128 ? 5 : 8;
  const int ctas = fit < 1 ? 1 : fit > regs ? regs : fit;
  const int most = 148 * ctas * kWarps / p.H;
  return p.B < 1 ? 1 : p.B < most ? p.B : most < 1 ? 1 : most;
}

template <typename T, int D, int KIND, bool BWD>
int launch(const DenseParams& p, cudaStream_t stream) {
  const bool table_grad = BWD && KIND != MF_BUCKETS_NONE && p.dbias_part;
  const int smem = smem_of(p, D, KIND, BWD, table_grad);
  SmallParams sp{p, slots_of(p, D, KIND, BWD, table_grad)};
  constexpr auto kernel = dense_attn_small_kernel<T, D, KIND, BWD>;
  constexpr int most = kWarps * (kTilesBytes<D, BWD> + small_table_bytes(KIND, kMaxBuckets) + (BWD && KIND != MF_BUCKETS_NONE ? (kMaxBuckets + 1) * 32 * 4 : 0));
  static_assert(most <= 227 * 1024, "");
  cudaError_t err = allow_shared<dense_attn_small_kernel<T, D, KIND, BWD>>(most);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  const long long warps = (long long)sp.slots * p.H;
  err = launch_dependent(kernel, dim3((unsigned)((warps + kWarps - 1) / kWarps)), dim3(kWarps * 32), smem, stream, sp);
  return err == cudaSuccess ? MF_OK : cuda_error(err, "dense attention of small entries");
}

template <typename T, bool BWD>
int pick(const DenseParams& p, int head_dim, int kind, cudaStream_t stream) {
  auto by_kind = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return kind == MF_BUCKETS_NONE     ? launch<T, D, MF_BUCKETS_NONE, BWD>(p, stream)
           : kind == MF_BUCKETS_OFFSET ? launch<T, D, MF_BUCKETS_OFFSET, BWD>(p, stream)
                                       : launch<T, D, MF_BUCKETS_PAIR, BWD>(p, stream);
  };
  return head_dim == 32   ? by_kind(std::integral_constant<int, 32>{})
         : head_dim == 64 ? by_kind(std::integral_constant<int, 64>{})
                          : by_kind(std::integral_constant<int, 128>{});
}

}  // namespace

bool dense_attn_small_applies(const DenseParams& p, bool backward) {
  return p.M >= 1 && p.N >= 1 && p.M <= kN && p.N <= kN && (!backward || p.H == p.K);
}
int dense_attn_small_slots(const DenseParams& p, int head_dim, int kind) { return slots_of(p, head_dim, kind, true, true); }
int dense_attn_small(const DenseParams& p, int dtype, int head_dim, int kind, bool backward, cudaStream_t stream) {
  if (backward) return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, true>(p, head_dim, kind, stream) : pick<__half, true>(p, head_dim, kind, stream);
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, false>(p, head_dim, kind, stream) : pick<__half, false>(p, head_dim, kind, stream);
}

}  // namespace mf
