// Dense attention of few queries on many keys (a token behind the keys that a sequence keeps): the keys of an entry in pieces, a CTA for each,
// joined by a second launch.
//
// All query heads that share a key head are rows of one 16-row tile (row = query * group + head of the group), so keys and values are
// read once for the group.  A warp takes every fourth tile of 16 keys of its CTA's piece through a ring of its own (cp.async, two tiles in
// flight while one is worked on, no barrier of the CTA), with a running maximum, sum and accumulator of its own; the warps meet in shared
// memory at the end, in their order.  Pieces are of one length for all entries, so that entries of different lengths balance; a second launch adds the
// pieces of a row in order.  Memory bounds it: a key and a value of 128 channels are 512 bytes for 64 products. 64 tokens behind 410 to 4096 keys,
// 32 heads on 8 of 128: 107 to 119 us, 5.0 to 5.5 TB/s; one behind 32771 keys 31 us, of which the pieces take 25 (5.4 TB/s).
#include "dense_attn.cuh"

namespace mf {
namespace {

constexpr int kTile = 16, kWarps = 4, kStages = 3, kThreads = kWarps * 32, kRows = 16;

struct SplitParams {
  DenseParams p;
  int pieces, piece;  // their number and length in keys, a multiple of kTile * kWarps
  float* acc;         // [entry * key head][row tile][piece][kRows][D], of unit scale exp2(-top)
  float* stat;        // the same without D: top, total
};

// Rows of D channels without padding: the 16-byte chunks of a row change places with its number, so that eight rows of one chunk lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t place(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (D == 32 ? (row >> 1) & 3 : row & 7)) << 4);
}
template <int D>
constexpr int kTileBytes = kTile * D * 2;
template <int D>
constexpr int kSplitSmem = kRows * D * 2 + kWarps * kStages * 2 * kTileBytes<D>;

template <typename T, int D, int KIND>
__global__ void __launch_bounds__(kThreads) dense_attn_split_kernel(const __grid_constant__ SplitParams sp) {
  const DenseParams& p = sp.p;
  constexpr int KS = D / 16, CHUNKS = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float meet[kWarps][kRows][2];
  float* table = reinterpret_cast<float*>(smem + kSplitSmem<D>);  // [min(group, kRows)][num_buckets + 1], the last entry for buckets beyond the table
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t s_q = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), s_kv = s_q + kRows * D * 2 + warp * kStages * 2 * kTileBytes<D>;
  const int group = p.H / p.K, rows = p.M * group, row_tiles = (rows + kRows - 1) / kRows, nb = p.num_buckets;
  launch_dependents();
  wait_for_previous();
  const int piece = blockIdx.x % sp.pieces, rt = blockIdx.x / sp.pieces % row_tiles, entry = blockIdx.x / sp.pieces / row_tiles;
  const int b = entry / p.K, kh = entry % p.K;
  const DenseLengths len = dense_lengths(p, b);
  const int row0 = rt * kRows, last_row = min(row0 + kRows, rows) - 1;
  // keys of this piece that some row sees
  const int from = piece * sp.piece, to = min(from + sp.piece, dense_limit(p, len, min(last_row / group, len.nq - 1)));
  const long long at = blockIdx.x;
  if (to <= from && sp.pieces > 1) {  // the join passes it by
    if (tid < kRows) sp.stat[(at * kRows + tid) * 2] = -INFINITY, sp.stat[(at * kRows + tid) * 2 + 1] = 0.f;
    return;
  }
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.key_mask_batch : nullptr;
  const int first = from + warp * kTile;  // of this warp's keys
  const int steps = to > first ? (to - first + kTile * kWarps - 1) / (kTile * kWarps) : 0;

  // this lane's chunks of a tile: rows lane / CHUNKS + it * (32 / CHUNKS), one column
  constexpr int ROWS_AT_ONCE = 32 / CHUNKS, ITS = kTile / ROWS_AT_ONCE;
  const int lane_row = lane / CHUNKS, lane_chunk = lane % CHUNKS;
  const T* k_src = static_cast<const T*>(p.k) + p.k_rows.at(b, kh, first + lane_row) + lane_chunk * 8;
  const T* v_src = static_cast<const T*>(p.v) + p.v_rows.at(b, kh, first + lane_row) + lane_chunk * 8;
  const T* any = static_cast<const T*>(p.k) + p.k_rows.at(b, kh, 0);  // where rows that are not read point
  auto load = [&](int t) {
    const uint32_t dst = s_kv + (t % kStages) * 2 * kTileBytes<D>;
    const long long k_at = (long long)t * kTile * kWarps * p.k_rows.token, v_at = (long long)t * kTile * kWarps * p.v_rows.token;
    const int key0 = first + t * kTile * kWarps;
    if (key0 + kTile <= to && !mask) {
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const uint32_t off = place<D>(lane_row + it * ROWS_AT_ONCE, lane_chunk);
        cp_async16(dst + off, k_src + k_at + it * ROWS_AT_ONCE * p.k_rows.token, true);
        cp_async16(dst + kTileBytes<D> + off, v_src + v_at + it * ROWS_AT_ONCE * p.v_rows.token, true);
      }
    } else {
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int key = key0 + lane_row + it * ROWS_AT_ONCE;
        const bool ok = key < to && (!mask || mask[key]);
        const uint32_t off = place<D>(lane_row + it * ROWS_AT_ONCE, lane_chunk);
        cp_async16(dst + off, ok ? k_src + k_at + it * ROWS_AT_ONCE * p.k_rows.token : any, ok);
        cp_async16(dst + kTileBytes<D> + off, ok ? v_src + v_at + it * ROWS_AT_ONCE * p.v_rows.token : any, ok);
      }
    }
  };
  for (int idx = tid; idx < kRows * CHUNKS; idx += kThreads) {
    const int r = idx / CHUNKS, c = idx % CHUNKS, row = row0 + r, i = row / group;
    const bool ok = row < rows && i < len.nq;
    cp_async16(s_q + place<D>(r, c), static_cast<const T*>(p.q) + (ok ? p.q_rows.at(b, kh * group + row % group, i) : 0) + c * 8, ok);
  }
  cp_async_commit();
#pragma unroll
  for (int t = 0; t < kStages - 1; ++t) {
    if (t < steps) load(t);
    cp_async_commit();
  }
  if (KIND != MF_BUCKETS_NONE)
    for (int i = tid; i < min(group, kRows) * (nb + 1); i += kThreads)
      table[i] = dense_bias_entry(p, i % (nb + 1), kh * group + (row0 + i / (nb + 1)) % group);

  int query[2], hi[2];
  const float* column[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e, row = row0 + r;
    query[e] = row / group;
    hi[e] = row < rows ? min(to, dense_limit(p, len, query[e])) : 0;
    column[e] = table + (group <= kRows ? r % group : r) * (nb + 1);  // the first column is of the head of row0
  }
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  const float sc2 = p.scale * kDenseLog2e;
  cp_async_wait<kStages - 1>();
  __syncthreads();  // the queries and the table
  uint32_t q_frag[KS][4];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) ldmatrix_x4(q_frag[ks], s_q + place<D>(lane & 15, ks * 2 + (lane >> 4)));

  for (int t = 0; t < steps; ++t) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // tile t is there for all lanes, and all are done with the stage of tile t - 1
    if (t + kStages - 1 < steps) load(t + kStages - 1);
    cp_async_commit();
    const uint32_t tile_k = s_kv + (t % kStages) * 2 * kTileBytes<D>, tile_v = tile_k + kTileBytes<D>;
    const int key0 = first + t * kTile * kWarps;
    uint32_t seen = 0xffffffffu;
    if (mask) seen = __ballot_sync(0xffffffffu, key0 + (lane & 15) < to && mask[min(key0 + (lane & 15), to - 1)] != 0);
    float s[2][4] = {}, s2[2][4] = {};  // two chains of products
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t w[4];
      ldmatrix_x4(w, tile_k + place<D>((lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1)));
      mma16816<T>(ks & 1 ? s2[0] : s[0], q_frag[ks], w[0], w[1]);
      mma16816<T>(ks & 1 ? s2[1] : s[1], q_frag[ks], w[2], w[3]);
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
          float z = (s[nt][2 * e + x] + s2[nt][2 * e + x]) * sc2;
          if (KIND != MF_BUCKETS_NONE && vis) {
            const int bucket = KIND == MF_BUCKETS_OFFSET ? dense_offset_bucket(p, key - query[e] - len.shift)
                                                         : p.buckets[b * p.bucket_batch + query[e] * p.bucket_row + key];
            z += column[e][min(bucket, nb)];
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
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {  // a maximum grew
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= alpha[e >> 1];
    }
    uint32_t a[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
      uint32_t w[4];
      ldmatrix_x4_trans(w, tile_v + place<D>((lane & 7) + ((lane >> 3) & 1) * 8, np * 2 + (lane >> 4)));
      mma16816<T>(acc[2 * np], a, w[0], w[1]);
      mma16816<T>(acc[2 * np + 1], a, w[2], w[3]);
    }
  }
  cp_async_wait<0>();

  // ---- the warps meet: each brings its rows to the common maximum, then the planes are added in order
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    total[e] += __shfl_xor_sync(0xffffffffu, total[e], 1);
    total[e] += __shfl_xor_sync(0xffffffffu, total[e], 2);
    if (t4 == 0) meet[warp][g + 8 * e][0] = top[e], meet[warp][g + 8 * e][1] = total[e];
  }
  __syncthreads();  // (and nobody reads a tile any more)
  float* plane = reinterpret_cast<float*>(smem);  // [kWarps][kRows][D]
  static_assert(kWarps * kRows * D * 4 <= kSplitSmem<D>, "");
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
  for (int idx = tid; idx < min(kRows, rows - row0) * (D / 4); idx += kThreads) {
    const int r = idx / (D / 4), c = idx % (D / 4) * 4, row = row0 + r;
    const float m = fmaxf(fmaxf(meet[0][r][0], meet[1][r][0]), fmaxf(meet[2][r][0], meet[3][r][0]));
    float l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      // (logits that are no numbers have no maximum, but a total that is none: whether something was seen is for the total to say)
      l += meet[w][r][0] == -INFINITY ? meet[w][r][1] : meet[w][r][1] * dense_exp2(meet[w][r][0] - m);
      const float4 x = *reinterpret_cast<const float4*>(plane + (w * kRows + r) * D + c);
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    if (sp.pieces == 1) {
      const int i = row / group, h = kh * group + row % group;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + p.out_rows.at(b, h, i) + c) =
          inv == 0.f ? make_uint2(0u, 0u) : make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
      if (p.lse && c == 0) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
    } else {
      *reinterpret_cast<float4*>(sp.acc + (at * kRows + r) * D + c) = v;
      if (c == 0) sp.stat[(at * kRows + r) * 2] = m, sp.stat[(at * kRows + r) * 2 + 1] = l;
    }
  }
}

// More than 32 pieces: a block per row, the pieces' weights into shared memory, then 128 / (D / 4) shares of the pieces, four channels to a thread, each share in order
// and the shares in order.
constexpr int kMostPieces = 320;
template <typename T, int D>
__global__ void __launch_bounds__(128) dense_attn_join_kernel(const __grid_constant__ SplitParams sp) {
  const DenseParams& p = sp.p;
  constexpr int SHARES = 128 / (D / 4);
  __shared__ float weight[kMostPieces];
  __shared__ float4 part[SHARES][D / 4];
  __shared__ float meet[4][2];
  launch_dependents();
  wait_for_previous();
  const int group = p.H / p.K, rows = p.M * group, row_tiles = (rows + kRows - 1) / kRows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x % rows, entry = blockIdx.x / rows, b = entry / p.K, kh = entry % p.K;
  const long long base = ((long long)entry * row_tiles + row / kRows) * sp.pieces;
  auto slot = [&](int s) { return (base + s) * kRows + row % kRows; };
  float m = -INFINITY;
  for (int s = tid; s < sp.pieces; s += 128) m = fmaxf(m, sp.stat[slot(s) * 2]);
  m = warp_max(m);
  if (lane == 0) meet[warp][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(meet[0][0], meet[1][0]), fmaxf(meet[2][0], meet[3][0]));
  float l = 0.f;
  for (int s = tid; s < sp.pieces; s += 128) {
    const float t = sp.stat[slot(s) * 2], w = t == -INFINITY ? 0.f : dense_exp2(t - m);
    weight[s] = w;
    l = fmaf(w, sp.stat[slot(s) * 2 + 1], l);  // (a weight of zero as well: a total that is no number stays none)
  }
  l = warp_sum(l);
  if (lane == 0) meet[warp][1] = l;
  __syncthreads();
  l = meet[0][1] + meet[1][1] + meet[2][1] + meet[3][1];
  const int share = tid / (D / 4), c = tid % (D / 4);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = share; s < sp.pieces; s += SHARES) {
    const float w = weight[s];
    if (w == 0.f) continue;  // (a piece without a key that the row sees wrote nothing)
    const float4 x = *reinterpret_cast<const float4*>(sp.acc + slot(s) * D + c * 4);
    sum.x = fmaf(w, x.x, sum.x), sum.y = fmaf(w, x.y, sum.y), sum.z = fmaf(w, x.z, sum.z), sum.w = fmaf(w, x.w, sum.w);
  }
  part[share][c] = sum;
  __syncthreads();
  if (share > 0) return;
#pragma unroll
  for (int x = 1; x < SHARES; ++x) {
    const float4 y = part[x][c];
    sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int i = row / group, h = kh * group + row % group;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + p.out_rows.at(b, h, i) + c * 4) =
      inv == 0.f ? make_uint2(0u, 0u) : make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
  if (p.lse && tid == 0) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
}

// Up to 32 pieces: a warp per row, a lane for the weight of each piece and D / 32 channels, the pieces in order.  (2048 rows of two pieces, with the walk over 512
// keys each: 13 us; with a block per row 17.)
template <typename T, int D>
__global__ void __launch_bounds__(128) dense_attn_join_few_kernel(const __grid_constant__ SplitParams sp, int total_rows) {
  const DenseParams& p = sp.p;
  constexpr int E = D / 32;
  launch_dependents();
  wait_for_previous();
  const int lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= total_rows) return;
  const int group = p.H / p.K, rows = p.M * group, row_tiles = (rows + kRows - 1) / kRows;
  const int row = at % rows, entry = at / rows, b = entry / p.K, kh = entry % p.K;
  const long long base = ((long long)entry * row_tiles + row / kRows) * sp.pieces;
  auto slot = [&](int s) { return (base + s) * kRows + row % kRows; };
  const float t = lane < sp.pieces ? sp.stat[slot(lane) * 2] : -INFINITY;
  const float m = warp_max(t), w = t == -INFINITY ? 0.f : dense_exp2(t - m);
  const float l = warp_sum(lane < sp.pieces ? w * sp.stat[slot(lane) * 2 + 1] : 0.f);  // (as above)
  float sum[E] = {};
#pragma unroll 4
  for (int s = 0; s < sp.pieces; ++s) {
    const float ws = __shfl_sync(~0u, w, s);
    if (ws == 0.f) continue;  // (a piece without a key that the row sees wrote nothing)
    const float* x = sp.acc + slot(s) * D + lane * E;
    float v[E];
    if constexpr (E == 4) {
      const float4 f = *reinterpret_cast<const float4*>(x);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else if constexpr (E == 2) {
      const float2 f = *reinterpret_cast<const float2*>(x);
      v[0] = f.x, v[1] = f.y;
    } else {
      v[0] = *x;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = fmaf(ws, v[e], sum[e]);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int i = row / group, h = kh * group + row % group;
  T* out = static_cast<T*>(p.out) + p.out_rows.at(b, h, i) + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = inv == 0.f ? 0.f : sum[e] * inv;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]));
  else if constexpr (E == 2) *reinterpret_cast<uint32_t*>(out) = pack2<T>(sum[0], sum[1]);
  else *out = from_f32<T>(sum[0]);
  if (p.lse && lane == 0) p.lse[((long long)b * p.H + h) * p.M + i] = l > 0.f || l != l ? m + log2f(l) : INFINITY;
}

struct Plan {
  int row_tiles, pieces, piece;
  long long blocks;
};
// Two CTAs fit an SM.  Few columns: one round of CTAs.  Many: some six rounds, which even out entries of different lengths.
Plan plan_of(const DenseParams& p) {
  constexpr int kUnit = kTile * kWarps;
  Plan plan;
  plan.row_tiles = (p.M * (p.H / p.K) + kRows - 1) / kRows;
  const long long columns = (long long)p.B * p.K * plan.row_tiles;
  long long piece = columns >= 148 ? (columns * p.N + 1775) / 1776 : (p.N + 296 / columns - 1) / (296 / columns);
  const long long least = columns >= 148 ? 512 : 128;
  piece = piece < least ? least : piece;
  plan.piece = (int)((piece + kUnit - 1) / kUnit * kUnit);
  plan.pieces = (p.N + plan.piece - 1) / plan.piece;
  if (plan.pieces < 1) plan.pieces = 1;
  plan.blocks = columns * plan.pieces;
  return plan;
}

template <typename T, int D>
int join(const SplitParams& sp, cudaStream_t stream) {
  const long long rows = (long long)sp.p.B * sp.p.H * sp.p.M;
  const cudaError_t err = sp.pieces <= 32 ? launch_dependent(dense_attn_join_few_kernel<T, D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, sp, (int)rows)
                                          : launch_dependent(dense_attn_join_kernel<T, D>, dim3((unsigned)rows), dim3(128), 0, stream, sp);
  return err == cudaSuccess ? MF_OK : cuda_error(err, "dense attention join");
}

template <typename T, int D, int KIND>
int launch(const DenseParams& p, void* workspace, cudaStream_t stream) {
  const Plan plan = plan_of(p);
  SplitParams sp{p, plan.pieces, plan.piece, static_cast<float*>(workspace), nullptr};
  sp.stat = sp.acc + plan.blocks * kRows * D;
  constexpr auto kernel = dense_attn_split_kernel<T, D, KIND>;
  const int group = p.H / p.K, smem = kSplitSmem<D> + (KIND == MF_BUCKETS_NONE ? 0 : (group < kRows ? group : kRows) * (p.num_buckets + 1) * 4);
  constexpr int most = kSplitSmem<D> + (KIND == MF_BUCKETS_NONE ? 0 : kRows * (kMaxBuckets + 1) * 4);
  cudaError_t err = allow_shared<dense_attn_split_kernel<T, D, KIND>>(most);
  if (err != cudaSuccess) return cuda_error(err, "dense attention shared memory");
  err = launch_dependent(kernel, dim3((unsigned)plan.blocks), dim3(kThreads), smem, stream, sp);
  if (err != cudaSuccess) return cuda_error(err, "dense attention of few queries");
  return plan.pieces > 1 ? join<T, D>(sp, stream) : MF_OK;
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

// Few rows to a key head, or few pairs in all, so that most SMs would stand idle through a long walk.  Microseconds here | on the better of the other families: one
// query, 8 heads of 64, 65 keys 3.3 | 5.2, 512 keys 5.8 | 9.8, 64 entries of 1024 keys 31 | 50.  8 heads of 64 (of 128 after the comma): 64 queries on 1024 keys 7.4 | 15.4,
// 10 | 18; 2^21 pairs: 256 on 1024 13 | 20, 15 | 21, 128 on 2048 13.3 | 13.5, 15 | 16, 64 on 4096 11 | 13, 16 | 16; 2^22 pairs: 256 on 2048 20 | 17, 22 | 20; 2^23:
// 64 on 16384 34 | 20, 34 | 24.  Heads of 32, which tcgen05 does not take: 72 tiles of 64 queries on 4096 keys 33 | 43.  Not measured on this side, since the rule
// leaves them to the others: batches of more than 16 rows to a key head (64 single tokens of 32 heads of 128 on one, behind 4096 keys, - | 435; the cache alone is 21).
bool dense_attn_split_applies(const DenseParams& p, int head_dim) {
  if (p.N <= 64 || p.N > (1 << 26)) return false;
  if ((long long)p.M * (p.H / p.K) <= kRows) return true;
  if (p.M > 256 || p.N < 512) return false;
  const long long rows = (long long)p.B * p.H * p.M;
  return rows * p.N <= 1 << 21 || (head_dim == 32 && p.N >= 2048 && (long long)p.B * p.H * ((p.M + 63) / 64) < 74);
}
size_t dense_attn_split_workspace_bytes(const DenseParams& p, int head_dim) {
  const Plan plan = plan_of(p);
  return plan.pieces > 1 ? dense_attn_join_bytes(p, head_dim, plan.pieces) : 0;
}
size_t dense_attn_join_bytes(const DenseParams& p, int head_dim, int pieces) {
  const long long row_tiles = ((long long)p.M * (p.H / p.K) + kRows - 1) / kRows;
  return align_up((size_t)p.B * p.K * row_tiles * pieces * kRows * (head_dim + 2) * sizeof(float), 256);
}
int dense_attn_join(const DenseParams& p, int dtype, int head_dim, int pieces, float* acc, float* stat, cudaStream_t stream) {
  const SplitParams sp{p, pieces, 0, acc, stat};
  if (dtype == MF_DTYPE_BF16) return head_dim == 64 ? join<__nv_bfloat16, 64>(sp, stream) : join<__nv_bfloat16, 128>(sp, stream);
  return head_dim == 64 ? join<__half, 64>(sp, stream) : join<__half, 128>(sp, stream);
}
int dense_attn_split(const DenseParams& p, int dtype, int head_dim, int kind, void* workspace, cudaStream_t stream) {
  return dtype == MF_DTYPE_BF16 ? pick<__nv_bfloat16>(p, head_dim, kind, workspace, stream) : pick<__half>(p, head_dim, kind, workspace, stream);
}

}  // namespace mf
