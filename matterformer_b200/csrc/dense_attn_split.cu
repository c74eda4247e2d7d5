// Dense attention of few queries on many keys (a token behind the keys that a sequence keeps): the keys of an entry in pieces, a CTA for each,
// joined by a second launch.
//
// All query heads that share a key head are rows of one 16-row tile (row = query * group + head of the group), so keys and values are
// read once for the group.  Tiles of 64 keys arrive by cp.async, four in flight; the four warps take 16 keys of a tile each, with a running maximum, sum
// and accumulator of their own, and meet in shared memory at the end in the order of the warps.  Pieces are of one length for all entries, so
// that entries of different lengths balance; the second launch adds the pieces of a row in order.  Memory bounds it: a key and a value of 128
// channels are 512 bytes for 64 products.
#include "dense_attn.cuh"

namespace mf {
namespace {

constexpr int kTile = 64, kStages = 4, kThreads = 128, kRows = 16;

struct SplitParams {
  DenseParams p;
  int pieces, piece;  // their number and length in keys, a multiple of kTile
  float* acc;         // [entry * key head][row tile][piece][kRows][D], of unit scale exp2(-top)
  float* stat;        // the same without D: top, total
};

template <int D>
constexpr int kSplitSmem = kRows * (D + 8) * 2 + kStages * 2 * kTile * (D + 8) * 2;

template <typename T, int D, int KIND>
__global__ void __launch_bounds__(kThreads) dense_attn_split_kernel(const __grid_constant__ SplitParams sp) {
  const DenseParams& p = sp.p;
  constexpr int LD = D + 8, TILE = kTile * LD * 2, KS = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float table[KIND == MF_BUCKETS_NONE ? 1 : kRows][KIND == MF_BUCKETS_NONE ? 1 : kTableEntries];
  __shared__ float meet[4][kRows][2];
  const uint32_t s_q = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), s_k = s_q + kRows * LD * 2, s_v = s_k + kStages * TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int group = p.H / p.K, rows = p.M * group, row_tiles = (rows + kRows - 1) / kRows;
  launch_dependents();
  wait_for_previous();
  const int piece = blockIdx.x % sp.pieces, rt = blockIdx.x / sp.pieces % row_tiles, entry = blockIdx.x / sp.pieces / row_tiles;
  const int b = entry / p.K, kh = entry % p.K;
  const DenseLengths len = dense_lengths(p, b);
  const int row0 = rt * kRows, last_row = min(row0 + kRows, rows) - 1;
  // keys of this piece that some row sees
  const int from = piece * sp.piece, to = min(from + sp.piece, dense_limit(p, len, min(last_row / group, len.nq - 1)));
  const int steps = to > from ? (to - from + kTile - 1) / kTile : 0;
  const long long at = blockIdx.x;
  if (steps == 0) {  // the join passes it by where nothing reaches it
    if (sp.pieces > 1 && tid < kRows) sp.stat[(at * kRows + tid) * 2] = -INFINITY, sp.stat[(at * kRows + tid) * 2 + 1] = 0.f;
    if (sp.pieces > 1) return;
  }
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.key_mask_batch : nullptr;
  const T* K = static_cast<const T*>(p.k) + p.k_rows.at(b, kh, 0);
  const T* V = static_cast<const T*>(p.v) + p.v_rows.at(b, kh, 0);

  auto load = [&](int t) {
    const int stage = t % kStages, key0 = from + t * kTile;
#pragma unroll
    for (int it = 0; it < kTile * (D / 8) / kThreads; ++it) {
      const int idx = it * kThreads + tid, r = idx / (D / 8), c = idx % (D / 8), key = key0 + r;
      const bool ok = key < to && (!mask || mask[key]);
      const uint32_t off = stage * TILE + (r * LD + c * 8) * 2;
      cp_async16(s_k + off, K + (ok ? key * p.k_rows.token : 0) + c * 8, ok);
      cp_async16(s_v + off, V + (ok ? key * p.v_rows.token : 0) + c * 8, ok);
    }
  };
  for (int idx = tid; idx < kRows * (D / 8); idx += kThreads) {
    const int r = idx / (D / 8), c = idx % (D / 8), row = row0 + r, i = row / group;
    const bool ok = row < rows && i < len.nq;
    cp_async16(s_q + (r * LD + c * 8) * 2, static_cast<const T*>(p.q) + (ok ? p.q_rows.at(b, kh * group + row % group, i) : 0) + c * 8, ok);
  }
#pragma unroll
  for (int t = 0; t < kStages - 1; ++t) {
    if (t < steps) load(t);
    cp_async_commit();
  }
  if (KIND != MF_BUCKETS_NONE)
    for (int i = tid; i < min(group, kRows) * kTableEntries; i += kThreads)
      table[i / kTableEntries][i % kTableEntries] = dense_bias_entry(p, i % kTableEntries, kh * group + (row0 + i / kTableEntries) % group);

  int query[2], hi[2], column[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = row0 + g + 8 * e;
    query[e] = row / group;
    hi[e] = row < rows ? min(to, dense_limit(p, len, query[e])) : 0;
    column[e] = group <= kRows ? (g + 8 * e) % group : g + 8 * e;  // of `table`, whose first is the head of row0
  }
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  const float sc2 = p.scale * kDenseLog2e;

  for (int t = 0; t < steps; ++t) {
    cp_async_wait<kStages - 2>();
    __syncthreads();  // tile t is there, and the stage of tile t - 1 is free
    if (t + kStages - 1 < steps) load(t + kStages - 1);
    cp_async_commit();
    const uint32_t off = (t % kStages) * TILE + warp * 16 * LD * 2;
    const int key0 = from + t * kTile + warp * 16;
    uint32_t seen = 0xffffffffu;
    if (mask) seen = __ballot_sync(0xffffffffu, key0 + (lane & 15) < to && mask[min(key0 + (lane & 15), to - 1)] != 0);
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t a[4], w[4];
      ldmatrix_x4(a, s_q + ((lane & 15) * LD + ks * 16 + (lane >> 4) * 8) * 2);
      ldmatrix_x4(w, s_k + off + (((lane & 7) + (lane >> 4) * 8) * LD + ks * 16 + ((lane >> 3) & 1) * 8) * 2);
      mma16816<T>(s[0], a, w[0], w[1]);
      mma16816<T>(s[1], a, w[2], w[3]);
    }
    float alpha[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float m = top[e];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int c = nt * 8 + 2 * t4 + x, key = key0 + c;
          const bool vis = key < hi[e] && ((seen >> c) & 1u);
          float z = s[nt][2 * e + x] * sc2;
          if (KIND != MF_BUCKETS_NONE && vis) {
            const int bucket = KIND == MF_BUCKETS_OFFSET ? dense_offset_bucket(p, key - query[e] - len.shift)
                                                         : p.buckets[b * p.bucket_batch + query[e] * p.bucket_row + key];
            z += table[column[e]][bucket];
          }
          z = vis ? z : -INFINITY;
          s[nt][2 * e + x] = z;
          m = fmaxf(m, z);
        }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float shift = m == -INFINITY ? 0.f : m;
      alpha[e] = dense_exp2(top[e] - shift);
      top[e] = m;
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) sum += s[nt][2 * e + x] = dense_exp2(s[nt][2 * e + x] - shift);
      total[e] = total[e] * alpha[e] + sum;
    }
    uint32_t a[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
      uint32_t w[4];
      ldmatrix_x4_trans(w, s_v + off + (((lane & 7) + ((lane >> 3) & 1) * 8) * LD + np * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[2 * np + h][e] *= alpha[e >> 1];
        mma16816<T>(acc[2 * np + h], a, w[2 * h], w[2 * h + 1]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- the warps meet: each brings its rows to the common maximum, then the planes are added in order
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    total[e] += __shfl_xor_sync(0xffffffffu, total[e], 1);
    total[e] += __shfl_xor_sync(0xffffffffu, total[e], 2);
    if (t4 == 0) meet[warp][g + 8 * e][0] = top[e], meet[warp][g + 8 * e][1] = total[e];
  }
  __syncthreads();
  float* plane = reinterpret_cast<float*>(smem);  // [4][kRows][D]
  static_assert(4 * kRows * D * 4 <= kSplitSmem<D>, "");
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e;
    const float m = fmaxf(fmaxf(meet[0][r][0], meet[1][r][0]), fmaxf(meet[2][r][0], meet[3][r][0]));
    const float mul = top[e] == -INFINITY ? 0.f : dense_exp2(top[e] - m);
#pragma unroll
    for (int nt = 0; nt < D / 8; ++nt)
      *reinterpret_cast<float2*>(plane + (warp * kRows + r) * D + nt * 8 + 2 * t4) = make_float2(acc[nt][2 * e] * mul, acc[nt][2 * e + 1] * mul);
  }
  __syncthreads();
  for (int idx = tid; idx < kRows * (D / 2); idx += kThreads) {
    const int r = idx / (D / 2), c = idx % (D / 2) * 2, row = row0 + r;
    const float m = fmaxf(fmaxf(meet[0][r][0], meet[1][r][0]), fmaxf(meet[2][r][0], meet[3][r][0]));
    float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      l += meet[w][r][0] == -INFINITY ? 0.f : meet[w][r][1] * dense_exp2(meet[w][r][0] - m);
      const float2 v = *reinterpret_cast<const float2*>(plane + (w * kRows + r) * D + c);
      x += v.x, y += v.y;
    }
    if (row >= rows) continue;
    if (sp.pieces == 1) {
      const int i = row / group, h = kh * group + row % group;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + p.out_rows.at(b, h, i) + c) = inv == 0.f ? 0u : pack2<T>(x * inv, y * inv);
      if (p.lse && c == 0) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
    } else {
      *reinterpret_cast<float2*>(sp.acc + (at * kRows + r) * D + c) = make_float2(x, y);
      if (c == 0) sp.stat[(at * kRows + r) * 2] = m, sp.stat[(at * kRows + r) * 2 + 1] = l;
    }
  }
}

// One warp per row: the pieces' weights, then their sum in order; a lane holds D / 32 channels.
template <typename T, int D>
__global__ void __launch_bounds__(128) dense_attn_join_kernel(const __grid_constant__ SplitParams sp) {
  const DenseParams& p = sp.p;
  launch_dependents();
  wait_for_previous();
  const int group = p.H / p.K, rows = p.M * group, row_tiles = (rows + kRows - 1) / kRows;
  const long long which = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (which >= (long long)p.B * p.K * rows) return;
  const int lane = threadIdx.x & 31, row = which % rows, entry = which / rows, b = entry / p.K, kh = entry % p.K;
  const long long base = ((long long)entry * row_tiles + row / kRows) * sp.pieces;
  const float* stat = sp.stat;
  const float* acc = sp.acc;
  auto slot = [&](int s) { return (base + s) * kRows + row % kRows; };
  float m = -INFINITY;
  for (int s = lane; s < sp.pieces; s += 32) m = fmaxf(m, stat[slot(s) * 2]);
  m = warp_max(m);
  constexpr int C = D / 32;
  float sum[C] = {}, l = 0.f;
  for (int s0 = 0; s0 < sp.pieces; s0 += 32) {
    const int mine = s0 + lane;
    const float t = mine < sp.pieces ? stat[slot(mine) * 2] : -INFINITY;
    const float w = t == -INFINITY ? 0.f : dense_exp2(t - m);
    const float part = w == 0.f ? 0.f : w * stat[slot(min(mine, sp.pieces - 1)) * 2 + 1];
#pragma unroll 4
    for (int s = 0; s < min(32, sp.pieces - s0); ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      l += __shfl_sync(0xffffffffu, part, s);
      if (ws == 0.f) continue;  // (a piece without a key that the row sees wrote nothing)
      const float* a = acc + slot(s0 + s) * D + lane * C;
#pragma unroll
      for (int c = 0; c < C; ++c) sum[c] = fmaf(ws, a[c], sum[c]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int i = row / group, h = kh * group + row % group;
  T* dst = static_cast<T*>(p.out) + p.out_rows.at(b, h, i) + lane * C;
#pragma unroll
  for (int c = 0; c < C; ++c) dst[c] = from_f32<T>(sum[c] * inv);
  if (p.lse && lane == 0) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
}

struct Plan {
  int row_tiles, pieces, piece;
  long long blocks;
};
// Some 1 200 CTAs (two on each SM, four times over) where the keys give as many pieces of at least 256.
Plan plan_of(const DenseParams& p) {
  Plan plan;
  plan.row_tiles = (p.M * (p.H / p.K) + kRows - 1) / kRows;
  const long long columns = (long long)p.B * p.K * plan.row_tiles;
  long long piece = (columns * p.N + 1183) / 1184;
  piece = piece < 256 ? 256 : piece;
  plan.piece = (int)((piece + kTile - 1) / kTile * kTile);
  plan.pieces = (p.N + plan.piece - 1) / plan.piece;
  if (plan.pieces < 1) plan.pieces = 1;
  plan.blocks = columns * plan.pieces;
  return plan;
}

template <typename T, int D, int KIND>
int launch(const DenseParams& p, void* workspace, cudaStream_t stream) {
  const Plan plan = plan_of(p);
  SplitParams sp{p, plan.pieces, plan.piece, static_cast<float*>(workspace), nullptr};
  sp.stat = sp.acc + plan.blocks * kRows * D;
  auto kernel = dense_attn_split_kernel<T, D, KIND>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem<D>);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  err = launch_dependent(kernel, dim3((unsigned)plan.blocks), dim3(kThreads), kSplitSmem<D>, stream, sp);
  if (err != cudaSuccess) return cuda_error(err, "dense attention of few queries");
  if (plan.pieces > 1) {
    const long long rows = (long long)p.B * p.H * p.M;
    err = launch_dependent(dense_attn_join_kernel<T, D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, sp);
    if (err != cudaSuccess) return cuda_error(err, "dense attention join");
  }
  return MF_OK;
}

template <typename T>
int pick(const DenseParams& p, int head_dim, int kind, void* workspace, cudaStream_t stream) {
  auto by_kind = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return kind == MF_BUCKETS_NONE     ? launch<T, D, MF_BUCKETS_NONE>(p, workspace, stream)
           : kind == MF_BUCKETS_OFFSET ? launch<T, D, MF_BUCKETS_OFFSET>(p, workspace, stream)
                                       : launch<T, D, MF_BUCKETS_PAIR>(p, workspace, stream);
  };
  return head_dim == 32   ? by_kind(std::integral_constant<int, 32>{})
         : head_dim == 64 ? by_kind(std::integral_constant<int, 64>{})
                          : by_kind(std::integral_constant<int, 128>{});
}

}  // namespace

// Few rows to a key head, or so few tiles of 64 queries that most SMs would stand idle through a long walk.
bool dense_attn_split_applies(const DenseParams& p) {
  if (p.N <= 64) return false;
  const long long tiles = (long long)p.B * p.H * ((p.M + 63) / 64);
  return (long long)p.M * (p.H / p.K) <= kRows || (p.N >= 512 && tiles < 74 && p.M <= 256);
}
size_t dense_attn_split_workspace_bytes(const DenseParams& p, int head_dim) {
  const Plan plan = plan_of(p);
  return plan.pieces > 1 ? align_up((size_t)plan.blocks * kRows * (head_dim + 2) * sizeof(float), 256) : 0;
}
int dense_attn_split(const DenseParams& p, int dtype, int head_dim, int kind, void* workspace, cudaStream_t stream) {
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16>(p, head_dim, kind, workspace, stream) : pick<__half>(p, head_dim, kind, workspace, stream);
}

}  // namespace mf
