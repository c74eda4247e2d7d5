// Entry points of dense attention with a learned bias by buckets, the sum of the table's gradient, and the buckets of a molecule's distances.
#include "dense_attn_sm100.cuh"

#include <string.h>

namespace mf {
namespace {

// dbias[bucket][head] = sum of the partial sums of all tiles of the head: a block for a head and 32 buckets, a warp for every 16th tile, the warps in
// order.  Sums in fp64: they are long and cancel.
constexpr int kSumWarps = 16;
__global__ void __launch_bounds__(kSumWarps * 32) bias_sum_kernel(const float* part, int B, int H, int tiles, int nb, void* out, int dtype) {
  launch_dependents();
  wait_for_previous();
  const int h = blockIdx.x % H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bucket = blockIdx.x / H * 32 + lane;
  const int n = B * tiles;
  double sum = 0.0;
  if (bucket < nb) {
#pragma unroll 8
    for (int i = warp; i < n; i += kSumWarps) {
      const int b = tiles == 1 ? i : i / tiles, t = i - b * tiles;
      sum += part[(((long long)b * H + h) * tiles + t) * nb + bucket];
    }
  }
  __shared__ double sums[kSumWarps][32];
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp > 0 || bucket >= nb) return;
  #pragma unroll
  for (int w = 1; w < kSumWarps; ++w) sum += sums[w][lane];
  const float v = (float)sum;
  const int at = bucket * H + h;
  if (dtype == MF_DTYPE_F32) static_cast<float*>(out)[at] = v;
  else if (dtype == MF_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[at] = from_f32<__nv_bfloat16>(v);
  else static_cast<__half*>(out)[at] = from_f32<__half>(v);
}

constexpr int kMaxEdges = kMaxBuckets - 1;
// Cells of squared distances: 64 to an octave (exponent and six bits of the mantissa), 16 octaves up to the last edge.
constexpr int kCells = 1024, kCellShift = 17;
struct Edges {
  double square[kMaxEdges];  // of the edges
  float low[kMaxEdges];      // the same in fp32
  alignas(4) uint8_t first[kCells];  // edges below a cell
  int base, n, zeros;  // zeros: edges of a distance of zero
};
__device__ __forceinline__ uint32_t param_word(const void* at) {
  uint32_t v;
  asm volatile("ld.u32 %0, [%1];" : "=r"(v) : "l"(at));
  return v;
}
constexpr float kDistanceError = 5e-7f;  // of a squared distance in fp32, in relation to it; 6 * 2^-24 and an edge's rounding
constexpr int kLeastSquare = 0x0d800000;  // 2^-100 as bits: below, its three squares may leave fp32's normal range, and that error does not hold

// A thread takes four columns, whose coordinates stay in registers, and walks over rows: `lanes` threads (a power of two up to 32) lie along a row, the rest
// of the block along the rows.  The squared distance is formed in fp32 (off by at most 6 * 2^-24 of itself, a sum of three squares); its leading bits name a cell, which
// knows the buckets below it and the one edge in it, if any: one load, one comparison.  A pair within that error of the edge, in a cell that several edges share
// or so near that squares leave fp32's range is decided in fp64, where the differences of fp32 coordinates are exact but for far apart exponents.
// What bounds it is instructions, some twenty a pair; two cells of 4096 atoms and 63 edges take 42.6 us (83 % of the issue slots; all pairs in fp64
// against all edges 463).
constexpr int kBucketThreads = 256, kBucketSteps = 16;
__global__ void __launch_bounds__(kBucketThreads) distance_buckets_kernel(const float* coords, const int32_t* num_atoms, int N, const __grid_constant__ Edges edges,
                                                                          uint8_t* out, long long batch_stride, long long row, int words, int lanes, int column_tiles,
                                                                          int row_tiles) {
  __shared__ float2 cells[kCells];  // the edge (infinity: none; not a number: several), the bucket below it as an integer
  launch_dependents();
  // (through generic addresses: loads of parameters go by the constant cache, one address of a warp after the other)
  for (int w = threadIdx.x; w < kCells / 4; w += kBucketThreads) {
    const uint32_t four = param_word(edges.first + 4 * w);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 4 * w + e, k = (four >> (8 * e)) & 255u;
      const float end = c == kCells - 1 ? INFINITY : __int_as_float(max(0, c + 1 + edges.base) << kCellShift) * (1.f + 2 * kDistanceError);
      const float one = k < edges.n ? __uint_as_float(param_word(edges.low + k)) : INFINITY;
      const float two = k + 1 < edges.n ? __uint_as_float(param_word(edges.low + k + 1)) : INFINITY;
      cells[c] = make_float2(c == 0 || c + edges.base <= (kLeastSquare >> kCellShift) || (k + 1 < edges.n && two <= end) ? __int_as_float(0x7fffffff) : one <= end ? one : INFINITY, __int_as_float(k));
    }
  }
  wait_for_previous();
  __syncthreads();
  const int ct = blockIdx.x % column_tiles, rt = blockIdx.x / column_tiles % row_tiles, b = blockIdx.x / column_tiles / row_tiles;
  const int n = num_atoms ? min(num_atoms[b], N) : N;
  const int at_once = kBucketThreads / lanes;
  const int j0 = (ct * lanes + (threadIdx.x & (lanes - 1))) * 4, i0 = rt * at_once * kBucketSteps + threadIdx.x / lanes;
  const float* x = coords + (long long)b * N * 3;
  float y[4][3];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int a = 0; a < 3; ++a) y[c][a] = j0 + c < n ? x[(j0 + c) * 3ll + a] : 0.f;
  const uint32_t there = j0 + 4 <= n ? ~0u : j0 < n ? (1u << (8 * (n - j0))) - 1u : 0u;  // bytes of columns that are atoms
  const int last = min(i0 + at_once * (kBucketSteps - 1), N - 1);
  const float* xi = x + i0 * 3ll;
  uint8_t* dst = out + b * batch_stride + i0 * row + j0;
  const uint8_t* at_cells = reinterpret_cast<const uint8_t*>(cells) - 8ll * edges.base;
  const int lowest = edges.base, highest = edges.base + kCells - 1;
#pragma unroll 2
  for (int i = i0; i <= last; i += at_once, xi += at_once * 3, dst += at_once * row) {
    uint32_t word = 0;
    if (i < n) {
      const float p0 = xi[0], p1 = xi[1], p2 = xi[2];
      uint32_t unsure = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float dx = p0 - y[c][0], dy = p1 - y[c][1], dz = p2 - y[c][2];
        const float d2 = fmaf(dz, dz, fmaf(dy, dy, dx * dx));
        const int cell = max(lowest, min(highest, __float_as_int(d2) >> kCellShift));
        const float2 e = *reinterpret_cast<const float2*>(at_cells + 8 * cell);
        const float past = d2 - e.x;
        if (!(fabsf(past) > d2 * kDistanceError)) unsure |= 255u << (8 * c);
        word |= (uint32_t)(__float_as_int(e.y) + (past >= 0.f)) << (8 * c);
      }
      unsure &= there;
      if (unsure) {
        word &= ~unsure;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          if (!((unsure >> (8 * c)) & 1u)) continue;
          const float* o = x + (j0 + c) * 3ll;
          const float q0 = o[0], q1 = o[1], q2 = o[2];
          int lo = 0, hi = edges.n;  // edges below lo are at or below the distance, those from hi on above it
          if (p0 == q0 && p1 == q1 && p2 == q2) {  // an atom and itself: every row has one
            lo = hi = (p0 - p0) + (p1 - p1) + (p2 - p2) == 0.f ? edges.zeros : 0;  // (at infinity that is no distance)
          } else {
            const double ex = (double)p0 - q0, ey = (double)p1 - q1, ez = (double)p2 - q2;
            const double e2 = __dadd_rn(__dadd_rn(__dmul_rn(ex, ex), __dmul_rn(ey, ey)), __dmul_rn(ez, ez));
            while (lo < hi) {
              const int mid = (lo + hi) / 2;
              if (e2 >= edges.square[mid]) lo = mid + 1;
              else hi = mid;
            }
          }
          word |= (uint32_t)lo << (8 * c);
        }
      }
      word &= there;
    }
    if (words) {  // rows that hold whole words, behind the last atom too
      if (j0 < row) *reinterpret_cast<uint32_t*>(dst) = word;
    } else {
      for (int c = 0; c < 4 && j0 + c < N; ++c) dst[c] = (uint8_t)(word >> (8 * c));
    }
  }
}

DenseRows rows_of(const MfRows& r) { return DenseRows{r.batch, r.head, r.token}; }

int check_rows(const char* name, const char* what, const void* base, const MfRows& r) {
  MF_CHECK_ALIGNED(name, base);
  MF_CHECK_ARG(r.batch % 8 == 0 && r.head % 8 == 0 && r.token % 8 == 0, "%s: strides of %s must be multiples of 8 elements, got %lld, %lld, %lld", name, what,
               (long long)r.batch, (long long)r.head, (long long)r.token);
  return MF_OK;
}

int check_args(const char* name, const MfDenseAttnArgs* a) {
  MF_CHECK_ARG(a != nullptr, "%s: args is NULL", name);
  MF_CHECK_ARG(a->dtype == MF_DTYPE_BF16 || a->dtype == MF_DTYPE_F16, "%s: dtype must be bf16 or fp16, got code %d", name, a->dtype);
  MF_CHECK_ARG(a->batch >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 && a->queries >= 0 && a->keys >= 0,
               "%s: heads must be a multiple of kv_heads and sizes not negative, got batch %d, heads %d, kv_heads %d, queries %d, keys %d", name, a->batch, a->heads,
               a->kv_heads, a->queries, a->keys);
  MF_CHECK_ARG(a->head_dim == 32 || a->head_dim == 64 || a->head_dim == 128, "%s: head_dim must be 32, 64 or 128, got %d", name, a->head_dim);
  MF_CHECK_ARG((long long)a->batch * a->heads * (((long long)(a->queries > a->keys ? a->queries : a->keys) + 63) / 64 + 1) < (1ll << 31) &&
                   a->queries < (1 << 30) && a->keys < (1 << 30),
               "%s: batch * heads * tiles of 64 rows must stay below 2^31 and lengths below 2^30", name);
  MF_CHECK_ARG(a->scale == a->scale && a->scale - a->scale == 0.f, "%s: scale must be finite", name);
  MF_CHECK_ARG(a->backend >= MF_DENSE_BACKEND_AUTO && a->backend <= MF_DENSE_BACKEND_TCGEN05, "%s: unknown backend %d", name, a->backend);
  const bool table = a->bias != nullptr;
  // (the buckets of no pairs have no address)
  const bool no_pairs = a->bucket_kind == MF_BUCKETS_PAIR && (a->batch == 0 || a->queries == 0 || a->keys == 0);
  MF_CHECK_ARG(table == (a->bucket_kind != MF_BUCKETS_NONE) && (table == (a->buckets != nullptr) || (table && no_pairs)), "%s: bias, buckets and bucket_kind go together", name);
  if (table) {
    MF_CHECK_ARG(a->bucket_kind == MF_BUCKETS_OFFSET || a->bucket_kind == MF_BUCKETS_PAIR, "%s: unknown bucket_kind %d", name, a->bucket_kind);
    MF_CHECK_ARG(a->num_buckets >= 1 && a->num_buckets <= kMaxBuckets, "%s: between 1 and %d buckets, got %d", name, kMaxBuckets, a->num_buckets);
    MF_CHECK_ARG(a->bias_dtype == MF_DTYPE_F32 || a->bias_dtype == MF_DTYPE_BF16 || a->bias_dtype == MF_DTYPE_F16, "%s: unknown bias_dtype %d", name, a->bias_dtype);
    MF_CHECK_ARG(a->bucket_kind != MF_BUCKETS_OFFSET || (a->reach >= 0 && a->reach < (1 << 30)), "%s: reach must lie between 0 and 2^30, got %d", name, a->reach);
    MF_CHECK_ARG(a->bucket_kind != MF_BUCKETS_PAIR || (a->bucket_row >= 0 && a->bucket_batch >= 0), "%s: strides of the buckets must not be negative", name);
  }
  if (a->batch == 0 || (a->queries == 0 && a->keys == 0)) return MF_OK;
  int rc;
  if ((a->queries > 0 && (MF_OK != (rc = check_rows(name, "q", a->q, a->q_rows)) || MF_OK != (rc = check_rows(name, "out", a->out, a->out_rows)))) ||
      (a->keys > 0 && (MF_OK != (rc = check_rows(name, "k", a->k, a->k_rows)) || MF_OK != (rc = check_rows(name, "v", a->v, a->v_rows)))))
    return rc;
  MF_CHECK_ARG((a->queries == 0 || (a->q && a->out)) && (a->keys == 0 || (a->k && a->v)), "%s: q, k, v and out must not be NULL", name);
  return MF_OK;
}

DenseParams params_of(const MfDenseAttnArgs& a) {
  DenseParams p{};
  p.q = a.q, p.k = a.k, p.v = a.v, p.grad_out = a.grad_out;
  p.out = a.out, p.dq = a.dq, p.dk = a.dk, p.dv = a.dv;
  p.q_rows = rows_of(a.q_rows), p.k_rows = rows_of(a.k_rows), p.v_rows = rows_of(a.v_rows), p.out_rows = rows_of(a.out_rows);
  p.go_rows = rows_of(a.grad_out_rows), p.dq_rows = rows_of(a.dq_rows), p.dk_rows = rows_of(a.dk_rows), p.dv_rows = rows_of(a.dv_rows);
  p.num_queries = a.num_queries, p.num_keys = a.num_keys, p.key_mask = a.key_mask, p.key_mask_batch = a.key_mask_batch;
  p.bias = a.bias, p.bias_dtype = a.bias_dtype, p.num_buckets = a.bias ? a.num_buckets : 0, p.reach = a.reach;
  p.buckets = a.buckets, p.bucket_batch = a.bucket_batch, p.bucket_row = a.bucket_row;
  p.lse = a.lse;
  p.B = a.batch, p.H = a.heads, p.K = a.kv_heads, p.M = a.queries, p.N = a.keys;
  p.causal = a.causal != 0, p.scale = a.scale;
  return p;
}

enum Family { kMma, kSmall, kSplit, kTensor };
// Where tiles of 128 rows on tcgen05 pay against warp-level tiles of 64 (microseconds on tcgen05 | warp-level, forward, then forward with backward, 8 heads, bias by the
// offset).  Head size 64: 64 x 256 tokens 39 | 57, 203 | 239; 64 x 200 tokens 43 | 54, 202 | 222; 42 x 384 tokens 52 | 75; 64 x 700 queries on 100 keys 85 | 89, 337 | 369;
// 8 x 64 queries on 1024 keys 17 | 25, 65 | 81 (64 of them 64 | 73, 326 | 289); but 85 x 192 tokens 53 | 46, 128 x 128 tokens 41 | 35, and equal from 257 to 300 tokens,
// where a third of a tile's rows is padding.  Head size 128: 64 x 256 tokens 55 | 99, 302 | 400; 64 x 700 queries on 100 keys 110 | 157, 511 | 604; 85 x 192 tokens 67 | 80
// forward, but 279 | 248 backward, and by pairs 76 | 67 forward.  There many short entries pay forward unless by pairs: 128 x 128 tokens 54 | 64, 128 x 65 tokens 51 | 54; few
// do not: 2 x 160 tokens 13 | 10.
// Fewer than 64 queries: 32 on 4096 keys, 32 heads of 64, 19 | 80, 91 | 185, four such entries 49 | 81, 251 | 266; but 16 entries of 17 on 2048 103 | 62, 512 | 380; heads of 128 122 |
// 137, 733 | 771.
bool tensor_pays(const DenseParams& p, int head_dim, int kind, bool backward) {
  if (p.N <= 64) return false;
  if (((p.M + 63ll) / 64) * ((p.N + 63ll) / 64) >= 16) return p.M >= 64 || head_dim == 128 || (long long)p.B * p.H <= 148;
  if (p.M < 64) return false;
  return !backward && head_dim == 128 && kind != MF_BUCKETS_PAIR && (long long)p.B * p.H >= 148;
}
Family fwd_family(const MfDenseAttnArgs& a, const DenseParams& p) {
  if (a.backend == MF_DENSE_BACKEND_MMA) return kMma;
  const bool takes = dense_tc_takes(p, a.head_dim, a.bucket_kind);
  if (a.backend == MF_DENSE_BACKEND_TCGEN05) return takes ? kTensor : kMma;
  return dense_attn_small_applies(p, false) ? kSmall : dense_attn_split_applies(p, a.head_dim) ? kSplit : takes && tensor_pays(p, a.head_dim, a.bucket_kind, false) ? kTensor : kMma;
}
Family bwd_family(const MfDenseAttnArgs& a, const DenseParams& p) {
  if (a.backend == MF_DENSE_BACKEND_MMA) return kMma;
  const bool takes = dense_tc_bwd_takes(p, a.head_dim, a.bucket_kind, a.bias && a.dbias);
  if (a.backend == MF_DENSE_BACKEND_TCGEN05) return takes ? kTensor : kMma;
  return dense_attn_small_applies(p, true) ? kSmall : takes && tensor_pays(p, a.head_dim, a.bucket_kind, true) ? kTensor : kMma;
}

// delta, then partial sums of the table's gradient for each head: as many as whichever of the tiled families runs needs.
struct BwdSpace {
  size_t part, total;
};
BwdSpace bwd_space(const MfDenseAttnArgs& a, const DenseParams& p) {
  BwdSpace s{};
  const bool small = bwd_family(a, p) == kSmall;
  s.part = small ? 0 : align_up((size_t)a.batch * a.heads * a.queries * sizeof(float), 256);
  auto most = [](size_t x, size_t y) { return x > y ? x : y; };
  const size_t sums = small ? dense_attn_small_slots(p, a.head_dim, a.bucket_kind) : most(dense_attn_mma_slots(p, a.head_dim), (size_t)a.batch * ((a.queries + kTcRows - 1) / kTcRows));
  s.total = s.part + (a.bias && a.dbias ? align_up(sums * a.heads * a.num_buckets * sizeof(float), 256) : 0);
  return s;
}

int check_space(const char* name, const MfDenseAttnArgs* a, size_t need) {
  if (need == 0) return MF_OK;
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("%s: %zu bytes of workspace needed, got %zu", name, need, a->workspace ? a->workspace_bytes : (size_t)0);
    return MF_ERR_WORKSPACE_TOO_SMALL;
  }
  MF_CHECK_ALIGNED(name, a->workspace);
  return MF_OK;
}

int forward(const char* name, const MfDenseAttnArgs* a, cudaStream_t stream, BoundedWaits waits) {
  const int rc = check_args(name, a);
  if (rc != MF_OK) return rc;
  if (a->batch == 0 || a->queries == 0) return MF_OK;
  const DenseParams p = params_of(*a);
  switch (fwd_family(*a, p)) {
    case kSmall: return dense_attn_small(p, a->dtype, a->head_dim, a->bucket_kind, false, stream);
    case kSplit: {
      const size_t need = dense_attn_split_workspace_bytes(p, a->head_dim);
      if (const int rc = check_space(name, a, need)) return rc;
      return dense_attn_split(p, a->dtype, a->head_dim, a->bucket_kind, a->workspace, stream);
    }
    case kTensor: {
      if (const int rc = check_space(name, a, dense_tc_fwd_workspace_bytes(p, a->head_dim))) return rc;
      return dense_attn_sm100_fwd(p, a->dtype, a->head_dim, a->bucket_kind, a->workspace, stream, waits);
    }
    default: return dense_attn_mma_fwd(p, a->dtype, a->head_dim, a->bucket_kind, stream);
  }
}

int backward(const char* name, const MfDenseAttnArgs* a, cudaStream_t stream, BoundedWaits waits) {
  int rc = check_args(name, a);
  if (rc != MF_OK) return rc;
  DenseParams p = params_of(*a);
  const bool table = a->bias && a->dbias;
  const BwdSpace space = a->batch ? bwd_space(*a, p) : BwdSpace{};
  if (MF_OK != (rc = check_space(name, a, space.total))) return rc;
  int entries = a->batch, tiles = 1;  // of partial sums for each head
  if (a->batch > 0) {
    MF_CHECK_ARG(a->queries == 0 || (a->grad_out && a->lse), "%s: grad_out and lse must not be NULL", name);
    if ((a->queries > 0 && MF_OK != (rc = check_rows(name, "grad_out", a->grad_out, a->grad_out_rows))) ||
        (a->dq && MF_OK != (rc = check_rows(name, "dq", a->dq, a->dq_rows))) || (a->dk && MF_OK != (rc = check_rows(name, "dk", a->dk, a->dk_rows))) ||
        (a->dv && MF_OK != (rc = check_rows(name, "dv", a->dv, a->dv_rows))))
      return rc;
    char* ws = static_cast<char*>(a->workspace);
    p.delta = reinterpret_cast<float*>(ws);
    if (table) p.dbias_part = reinterpret_cast<float*>(ws + space.part);
    DenseTcParams tc{p, {}, {}, {}, {}, waits};
    Family family = bwd_family(*a, p);
    if (family == kTensor && !dense_tc_maps(tc, a->dtype, a->head_dim, true)) family = kMma;
    switch (family) {
      case kSmall:
        entries = dense_attn_small_slots(p, a->head_dim, a->bucket_kind), tiles = 1;
        rc = dense_attn_small(p, a->dtype, a->head_dim, a->bucket_kind, true, stream);
        break;
      case kTensor:
        tiles = (a->queries + kTcRows - 1) / kTcRows;
        rc = dense_attn_sm100_bwd(tc, a->dtype, a->head_dim, a->bucket_kind, stream);
        break;
      default:
        entries = dense_attn_mma_slots(p, a->head_dim);
        rc = dense_attn_mma_bwd(p, a->dtype, a->head_dim, a->bucket_kind, stream);
    }
    if (rc != MF_OK) return rc;
  }
  if (!table) return MF_OK;
  const cudaError_t err = launch_dependent(bias_sum_kernel, dim3(a->heads * ((a->num_buckets + 31) / 32)), dim3(kSumWarps * 32), 0, stream, p.dbias_part, entries, a->heads, tiles,
                                           a->num_buckets, a->dbias, a->bias_dtype);
  return err == cudaSuccess ? MF_OK : cuda_error(err, "dense attention table gradient");
}

// The last expired wait of the forward kernels, or of the backward ones.
int take_status(int word, int32_t* host_status, cudaStream_t stream) {
  int32_t fwd = 0, bwd = 0;
  int rc = dense_attn_take_fwd_status(word, &fwd, stream);
  if (rc == MF_OK) rc = dense_attn_take_bwd_status(word, &bwd, stream);
  *host_status = fwd ? fwd : bwd;
  return rc;
}

}  // namespace
}  // namespace mf

extern "C" {

size_t mf_dense_attn_fwd_workspace_bytes(const MfDenseAttnArgs* a) {
  using namespace mf;
  if (check_args("mf_dense_attn_fwd_workspace_bytes", a) != MF_OK || a->batch == 0 || a->queries == 0) return 0;
  const DenseParams p = params_of(*a);
  const Family family = fwd_family(*a, p);
  return family == kSplit ? dense_attn_split_workspace_bytes(p, a->head_dim) : family == kTensor ? dense_tc_fwd_workspace_bytes(p, a->head_dim) : 0;
}
size_t mf_dense_attn_bwd_workspace_bytes(const MfDenseAttnArgs* a) {
  using namespace mf;
  if (check_args("mf_dense_attn_bwd_workspace_bytes", a) != MF_OK || a->batch == 0) return 0;
  return bwd_space(*a, params_of(*a)).total;
}

int mf_dense_attn_fwd(const MfDenseAttnArgs* a, void* stream) { return mf::forward("mf_dense_attn_fwd", a, static_cast<cudaStream_t>(stream), {}); }
int mf_dense_attn_bwd(const MfDenseAttnArgs* a, void* stream) { return mf::backward("mf_dense_attn_bwd", a, static_cast<cudaStream_t>(stream), {}); }

int mf_dense_attn_status(int32_t* host_status, void* stream) {
  MF_CHECK_ARG(host_status != nullptr, "mf_dense_attn_status: null pointer");
  return mf::take_status(0, host_status, static_cast<cudaStream_t>(stream));
}
int mf_selftest_dense_attn_give_up(const MfDenseAttnArgs* a, int32_t backward, int32_t kind, int64_t limit_cycles, int32_t* host_status, void* stream_) {
  using namespace mf;
  const char* name = "mf_selftest_dense_attn_give_up";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  MF_CHECK_ARG(a && kind >= 0 && kind <= 4 && a->backend == MF_DENSE_BACKEND_TCGEN05, "%s: bad argument", name);
  MF_CHECK_ARG(limit_cycles >= 10000 && limit_cycles <= kWaitLimitCycles, "%s: the limit must lie in [10^4, 2^31] clocks", name);
  BoundedWaits waits;
  waits.limit = limit_cycles, waits.withheld = kind, waits.word = host_status != nullptr;
  const int rc = backward ? mf::backward(name, a, stream, waits) : forward(name, a, stream, waits);
  return rc != MF_OK || !host_status ? rc : take_status(1, host_status, stream);
}

int mf_distance_buckets(const float* coords, const int32_t* num_atoms, int32_t batch, int32_t tokens, const double* edges, int32_t num_edges, uint8_t* buckets,
                        int64_t batch_stride, int64_t row, void* stream) {
  using namespace mf;
  const char* name = "mf_distance_buckets";
  int lanes = 32;
  while (lanes > 1 && lanes / 2 * 4 >= tokens) lanes /= 2;
  const int at_once = kBucketThreads / lanes * kBucketSteps, column_tiles = (int)((tokens + lanes * 4ll - 1) / (lanes * 4)), row_tiles = (int)((tokens + at_once - 1ll) / at_once);
  const long long tiles = (long long)column_tiles * row_tiles * batch;
  MF_CHECK_ARG(batch >= 0 && tokens >= 0 && tokens <= 1 << 20 && tiles < (1ll << 31), "%s: sizes out of range: %d molecules of %d atoms", name, batch, tokens);
  MF_CHECK_ARG(num_edges >= 0 && num_edges <= kMaxEdges && (num_edges == 0 || edges), "%s: at most %d edges, got %d", name, kMaxEdges, num_edges);
  Edges e{};
  for (int i = 0; i < num_edges; ++i) {
    MF_CHECK_ARG(edges[i] >= 0.0 && (i == 0 || edges[i] >= edges[i - 1]), "%s: edges must ascend from 0 on", name);
    e.square[i] = edges[i] * edges[i];
    e.low[i] = (float)e.square[i];
  }
  e.n = num_edges;
  while (e.zeros < num_edges && e.square[e.zeros] == 0.0) ++e.zeros;
  auto bits = [](float f) { int i; memcpy(&i, &f, 4); return i; };
  auto value = [](int i) { float f; memcpy(&f, &i, 4); return f; };
  const float least = value(kLeastSquare), last = num_edges && e.low[num_edges - 1] > least ? e.low[num_edges - 1] : least;
  e.base = (bits(last) >> kCellShift) - (kCells - 2);
  for (int c = 0, k = 0; c < kCells; ++c) {  // what the table says is where the search begins: too low costs time alone
    const long long start = (long long)(c + e.base) * (1 << kCellShift);
    const int at = start > 0x7f000000ll ? 0x7f000000 : start > 0 ? (int)start : 0;
    while (c > 0 && k < num_edges && at > 0 && e.low[k] < value(at) * (1.f - 2 * kDistanceError)) ++k;
    e.first[c] = (uint8_t)k;
  }
  if (batch == 0 || tokens == 0) return MF_OK;
  MF_CHECK_ARG(coords && buckets && row >= tokens && batch_stride >= (int64_t)(tokens - 1) * row + tokens, "%s: rows of the buckets must hold %d entries", name, tokens);
  // (rows of the call's own, by the contract: a word each, the last columns' too; 1024 molecules of 29 atoms 6.2 us, with those byte by byte 6.4)
  const int words = row % 4 == 0 && batch_stride % 4 == 0 && batch_stride >= tokens * row && reinterpret_cast<uintptr_t>(buckets) % 4 == 0;
  const cudaError_t err = launch_dependent(distance_buckets_kernel, dim3((unsigned)tiles), dim3(kBucketThreads), 0, static_cast<cudaStream_t>(stream), coords, num_atoms,
                                           tokens, e, buckets, batch_stride, row, words, lanes, column_tiles, row_tiles);
  return err == cudaSuccess ? MF_OK : cuda_error(err, name);
}

}  // extern "C"
