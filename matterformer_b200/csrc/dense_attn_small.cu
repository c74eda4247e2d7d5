// Dense attention with a learned bias by buckets on at most 32 queries and 32 keys (small molecules): a warp for every (entry, head), its logits, probabilities
// and their gradients whole in registers.
//
// The operands of an item are 32 rows each in the warp's own part of shared memory (cp.async in, 16-byte rows out, both coalesced); nothing is
// shared between warps, so they drift apart and hide each other's latencies.  A row of the softmax lies in four lanes: its maximum, sum and, backward,
// delta = sum_j p_j dP_j are exact sums of what the warp holds, and `out` is not read again.  P and dS are transposed in 8 x 8 tiles
// (movmatrix) where a product runs over the queries.  Warps stay with one head and walk over the entries, so the table's gradient is summed per
// lane in shared memory over the whole walk and leaves once.  Memory bounds both passes: an item of 29 tokens and 64 channels is 15 KB forward, 26 KB
// backward, for 1.7 and 4.3 MFLOP with the padding.
#include "dense_attn.cuh"

namespace mf {
namespace {

constexpr int kWarps = 4, kN = 32;

template <int D>
constexpr int kTile = kN * (D + 8) * 2;

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// rows [0, n) of a head into the warp's tile, zeros behind them and where `mask` is zero
template <typename T, int D>
__device__ __forceinline__ void rows_in(uint32_t tile, const T* src, long long stride, int n, uint32_t shown, int lane) {
#pragma unroll
  for (int it = 0; it < kN * (D / 8) / 32; ++it) {
    const int idx = it * 32 + lane, r = idx / (D / 8), c = idx % (D / 8);
    const bool ok = r < n && ((shown >> r) & 1u);
    cp_async16(tile + (r * (D + 8) + c * 8) * 2, src + (ok ? r * stride : 0) + c * 8, ok);
  }
}
template <typename T, int D>
__device__ __forceinline__ void rows_out(T* dst, long long stride, int rows, const uint8_t* tile, int lane) {
#pragma unroll
  for (int it = 0; it < kN * (D / 8) / 32; ++it) {
    const int idx = it * 32 + lane, r = idx / (D / 8), c = idx % (D / 8);
    if (r < rows) *reinterpret_cast<uint4*>(dst + r * stride + c * 8) = *reinterpret_cast<const uint4*>(tile + (r * (D + 8) + c * 8) * 2);
  }
}
// a 16 x D accumulator into rows [row0, row0 + 16) of a tile; a factor of zero gives zeros whatever was summed
template <typename T, int D>
__device__ __forceinline__ void keep(uint8_t* tile, int row0, const float (&acc)[D / 8][4], float m0, float m1, int lane) {
  const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int nt = 0; nt < D / 8; ++nt) {
    *reinterpret_cast<uint32_t*>(tile + ((row0 + g) * (D + 8) + nt * 8 + 2 * t4) * 2) = m0 == 0.f ? 0u : pack2<T>(acc[nt][0] * m0, acc[nt][1] * m0);
    *reinterpret_cast<uint32_t*>(tile + ((row0 + g + 8) * (D + 8) + nt * 8 + 2 * t4) * 2) = m1 == 0.f ? 0u : pack2<T>(acc[nt][2] * m1, acc[nt][3] * m1);
  }
}
// s (16 x 32) = rows [row0, row0 + 16) of tile a . rows of tile b
template <typename T, int D>
__device__ __forceinline__ void product(float (&s)[4][4], uint32_t a_tile, int row0, uint32_t b_tile, bool both, int lane) {
  constexpr int LD = D + 8;
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    uint32_t a[4], w[4];
    ldmatrix_x4(a, a_tile + ((row0 + (lane & 15)) * LD + ks * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
    for (int np = 0; np < 2; ++np) {
      if (np == 1 && !both) continue;
      ldmatrix_x4(w, b_tile + ((np * 16 + (lane & 7) + (lane >> 4) * 8) * LD + ks * 16 + ((lane >> 3) & 1) * 8) * 2);
      mma16816<T>(s[2 * np], a, w[0], w[1]);
      mma16816<T>(s[2 * np + 1], a, w[2], w[3]);
    }
  }
}
// acc (16 x D) = a (16 x 32, packed) . rows of tile b
template <typename T, int D>
__device__ __forceinline__ void contract(float (&acc)[D / 8][4], const uint32_t (&a)[2][4], uint32_t b_tile, bool both, int lane) {
#pragma unroll
  for (int nt = 0; nt < D / 8; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    if (kk == 1 && !both) continue;
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
      uint32_t w[4];
      ldmatrix_x4_trans(w, b_tile + ((kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * (D + 8) + np * 16 + (lane >> 4) * 8) * 2);
      mma16816<T>(acc[2 * np], a[kk], w[0], w[1]);
      mma16816<T>(acc[2 * np + 1], a[kk], w[2], w[3]);
    }
  }
}

struct SmallParams {
  DenseParams p;
  int slots;  // warps of a head
};

template <int D, bool BWD>
constexpr int kSmallSmem = kWarps * (BWD ? 4 : 3) * kTile<D>;

template <typename T, int D, int KIND, bool BWD>
__global__ void __launch_bounds__(kWarps * 32) dense_attn_small_kernel(const __grid_constant__ SmallParams sp) {
  const DenseParams& p = sp.p;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  // tiles of the warp: Q K V (dO); then every warp's column of the table, then its sums
  uint8_t* mine = smem + warp * (BWD ? 4 : 3) * kTile<D>;
  uint8_t *t_q = mine, *t_k = mine + kTile<D>, *t_v = mine + 2 * kTile<D>, *t_o = mine + 3 * kTile<D>;
  const uint32_t s_q = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), s_k = s_q + kTile<D>, s_v = s_k + kTile<D>, s_o = s_v + kTile<D>;
  float* table = reinterpret_cast<float*>(smem + kSmallSmem<D, BWD>) + warp * kTableEntries;
  const int nb = p.num_buckets;
  float* sums = reinterpret_cast<float*>(smem + kSmallSmem<D, BWD>) + kWarps * kTableEntries + warp * (nb + 1) * 32 + lane;
  const bool table_grad = BWD && KIND != MF_BUCKETS_NONE && p.dbias_part;
  launch_dependents();
  wait_for_previous();

  const int id = blockIdx.x * kWarps + warp, h = id % p.H, slot = id / p.H;
  if (slot >= sp.slots) return;
  const int kh = h / (p.H / p.K);
  if (KIND != MF_BUCKETS_NONE)
    for (int i = lane; i < kTableEntries; i += 32) table[i] = dense_bias_entry(p, i, h);
  if (table_grad)
    for (int i = 0; i <= nb; ++i) sums[i * 32] = 0.f;
  const float sc2 = p.scale * kDenseLog2e;

  for (int b = slot; b < p.B; b += sp.slots) {
    const DenseLengths len = dense_lengths(p, b);
    uint32_t shown = 0xffffffffu;
    if (p.key_mask) shown = __ballot_sync(0xffffffffu, lane < p.N && p.key_mask[b * p.key_mask_batch + lane] != 0);
    rows_in<T, D>(s_q, static_cast<const T*>(p.q) + p.q_rows.at(b, h, 0), p.q_rows.token, len.nq, 0xffffffffu, lane);
    rows_in<T, D>(s_k, static_cast<const T*>(p.k) + p.k_rows.at(b, kh, 0), p.k_rows.token, len.nk, shown, lane);
    rows_in<T, D>(s_v, static_cast<const T*>(p.v) + p.v_rows.at(b, kh, 0), p.v_rows.token, len.nk, shown, lane);
    if (BWD) rows_in<T, D>(s_o, static_cast<const T*>(p.grad_out) + p.go_rows.at(b, h, 0), p.go_rows.token, len.nq, 0xffffffffu, lane);
    cp_async_commit();

    // visible keys of the thread's four rows (g, g + 8, g + 16, g + 24) as bits, their buckets, a byte each
    uint32_t see[4], bucket[KIND == MF_BUCKETS_NONE ? 1 : 8];
    float lse[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = g + 8 * x, limit = dense_limit(p, len, i);
      see[x] = (limit >= 32 ? 0xffffffffu : (1u << limit) - 1u) & shown;
      if (BWD) lse[x] = i < len.nq ? p.lse[((long long)b * p.H + h) * p.M + i] : INFINITY;
    }
    if (KIND != MF_BUCKETS_NONE) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int nt = 0; nt < 4; nt += 2) {
          uint32_t word = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int i = g + 8 * x, j = (nt + (y >> 1)) * 8 + 2 * t4 + (y & 1);
            uint32_t v = 0;
            if ((see[x] >> j) & 1u)
              v = KIND == MF_BUCKETS_OFFSET ? dense_offset_bucket(p, j - i - len.shift) : p.buckets[b * p.bucket_batch + i * p.bucket_row + j];
            word |= v << (8 * y);
          }
          bucket[2 * x + (nt >> 1)] = word;
        }
    }
    auto bucket_of = [&](int x, int nt, int e) { return (int)((bucket[2 * x + (nt >> 1)] >> (16 * (nt & 1) + 8 * e)) & 255u); };
    const bool q2 = len.nq > 16, k2 = len.nk > 16;
    cp_async_wait<0>();
    __syncwarp();

    uint32_t P[2][2][4], S[BWD ? 2 : 1][2][4];  // packed, [query half][key half]: A operands of products over the keys
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
      product<T, D>(s, s_q, mt * 16, s_k, k2, lane);
      if constexpr (BWD) product<T, D>(dp, s_o, mt * 16, s_v, k2, lane);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 2 * mt + x;
        float m = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float z = s[nt][2 * x + e] * sc2;
            if (KIND != MF_BUCKETS_NONE) z += table[bucket_of(row, nt, e)];
            z = (see[row] >> (nt * 8 + 2 * t4 + e)) & 1u ? z : -INFINITY;
            s[nt][2 * x + e] = z;
            m = fmaxf(m, z);
          }
        if constexpr (!BWD) {
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float shift = m == -INFINITY ? 0.f : m;
          float l = 0.f;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) l += s[nt][2 * x + e] = dense_exp2(s[nt][2 * x + e] - shift);
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const int i = mt * 16 + g + 8 * x;
          if (p.lse && t4 == 0 && i < p.M) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
          lse[row] = l > 0.f || l != l ? 1.f / l : 0.f;
        } else {
          float d = 0.f;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float z = s[nt][2 * x + e], pr = z == -INFINITY ? 0.f : dense_exp2(z - lse[row]);
              s[nt][2 * x + e] = pr;
              if (pr != 0.f) d = fmaf(pr, dp[nt][2 * x + e], d);
            }
          d += __shfl_xor_sync(0xffffffffu, d, 1);
          d += __shfl_xor_sync(0xffffffffu, d, 2);
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float pr = s[nt][2 * x + e];
              dp[nt][2 * x + e] = pr == 0.f ? 0.f : pr * (dp[nt][2 * x + e] - d);
            }
          if (table_grad) {  // a column of sums for every lane: no two threads meet in one
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if ((see[row] >> (nt * 8 + 2 * t4 + e)) & 1u) sums[min(bucket_of(row, nt, e), nb) * 32] += dp[nt][2 * x + e];
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
        contract<T, D>(acc, P[mt], s_v, k2, lane);
        keep<T, D>(t_q, mt * 16, acc, mt && !q2 ? 0.f : lse[2 * mt], mt && !q2 ? 0.f : lse[2 * mt + 1], lane);
      }
      if (!q2 && p.lse && t4 == 0)
#pragma unroll
        for (int x = 2; x < 4; ++x)
          if (g + 8 * x < p.M) p.lse[((long long)b * p.H + h) * p.M + g + 8 * x] = INFINITY;
      __syncwarp();
      rows_out<T, D>(static_cast<T*>(p.out) + p.out_rows.at(b, h, 0), p.out_rows.token, p.M, t_q, lane);
    } else {
      __syncwarp();  // the values have been read
      if (p.dq) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          if (mt == 1 && p.M <= 16) continue;
          contract<T, D>(acc, S[mt], s_k, k2, lane);
          keep<T, D>(t_v, mt * 16, acc, mt * 16 + g < len.nq ? p.scale : 0.f, mt * 16 + g + 8 < len.nq ? p.scale : 0.f, lane);
        }
        __syncwarp();  // and the keys
        rows_out<T, D>(static_cast<T*>(p.dq) + p.dq_rows.at(b, h, 0), p.dq_rows.token, p.M, t_v, lane);
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
          if (kk == 1 && p.N <= 16) continue;
          turned(a, P, kk);
          contract<T, D>(acc, a, s_o, q2, lane);
          keep<T, D>(t_k, kk * 16, acc, real(kk * 16 + g) ? 1.f : 0.f, real(kk * 16 + g + 8) ? 1.f : 0.f, lane);
        }
        __syncwarp();
        rows_out<T, D>(static_cast<T*>(p.dv) + p.dv_rows.at(b, kh, 0), p.dv_rows.token, p.N, t_k, lane);
      }
      if (p.dk) {
        __syncwarp();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          if (kk == 1 && p.N <= 16) continue;
          turned(a, S, kk);
          contract<T, D>(acc, a, s_q, q2, lane);
          keep<T, D>(t_o, kk * 16, acc, real(kk * 16 + g) ? p.scale : 0.f, real(kk * 16 + g + 8) ? p.scale : 0.f, lane);
        }
        __syncwarp();
        rows_out<T, D>(static_cast<T*>(p.dk) + p.dk_rows.at(b, kh, 0), p.dk_rows.token, p.N, t_o, lane);
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

// Warps of a head: as many as fit the chip at `ctas` to an SM, at most one for each entry.
int slots_of(const DenseParams& p, int ctas) {
  const int most = 148 * ctas * kWarps / p.H;
  return p.B < 1 ? 1 : p.B < most ? p.B : most < 1 ? 1 : most;
}
int smem_of(const DenseParams& p, int head_dim, bool bwd, bool table_grad) {
  const int tiles = kWarps * (bwd ? 4 : 3) * kN * (head_dim + 8) * 2;
  return tiles + (p.bias ? kWarps * kTableEntries * 4 : 0) + (table_grad ? kWarps * (p.num_buckets + 1) * 32 * 4 : 0);
}
int ctas_of(const DenseParams& p, int head_dim, bool bwd, bool table_grad) {
  const int fit = 227 * 1024 / (smem_of(p, head_dim, bwd, table_grad) + 1024);
  return fit < 1 ? 1 : fit > 4 ? 4 : fit;
}

template <typename T, int D, int KIND, bool BWD>
int launch(const DenseParams& p, cudaStream_t stream) {
  const bool table_grad = BWD && KIND != MF_BUCKETS_NONE && p.dbias_part;
  const int smem = smem_of(p, D, BWD, table_grad);
  SmallParams sp{p, slots_of(p, ctas_of(p, D, BWD, table_grad))};
  auto kernel = dense_attn_small_kernel<T, D, KIND, BWD>;
  constexpr int most = kSmallSmem<D, BWD> + kWarps * kTableEntries * 4 + (BWD ? kWarps * (kMaxBuckets + 1) * 32 * 4 : 0);
  static_assert(most <= 227 * 1024, "");
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
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
int dense_attn_small_slots(const DenseParams& p, int head_dim) { return slots_of(p, ctas_of(p, head_dim, true, true)); }
int dense_attn_small(const DenseParams& p, int dtype, int head_dim, int kind, bool backward, cudaStream_t stream) {
  if (backward) return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, true>(p, head_dim, kind, stream) : pick<__half, true>(p, head_dim, kind, stream);
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16, false>(p, head_dim, kind, stream) : pick<__half, false>(p, head_dim, kind, stream);
}

}  // namespace mf
