// Entry points of dense attention with a learned bias by buckets, the sum of the table's gradient, and the buckets of a molecule's distances.
#include "dense_attn.cuh"

namespace mf {
namespace {

// dbias[bucket][head] = sum of the partial sums of all tiles of the head, over batch entries and tiles in order; a block for every (head, bucket),
// sums in fp64 (they are long and cancel)
__global__ void __launch_bounds__(128) bias_sum_kernel(const float* part, int B, int H, int tiles, int nb, void* out, int dtype) {
  const int h = blockIdx.x % H, bucket = blockIdx.x / H;
  const long long n = (long long)B * tiles;
  double sum = 0.0;
  for (long long i = threadIdx.x; i < n; i += 128) sum += part[((i / tiles * H + h) * tiles + i % tiles) * nb + bucket];
  __shared__ double sums[128];
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 64; o > 0; o >>= 1) {
    if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float v = (float)sums[0];
    const int at = bucket * H + h;
    if (dtype == MF_DTYPE_F32) static_cast<float*>(out)[at] = v;
    else if (dtype == MF_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[at] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(out)[at] = from_f32<__half>(v);
  }
}

constexpr int kMaxEdges = kMaxBuckets - 1;
struct Edges {
  double square[kMaxEdges];
};

// One thread per pair.  The squared distance is formed in fp64, where the differences of fp32 coordinates are exact but for far apart exponents,
// so that a pair next to an edge falls on the side that it belongs to.
__global__ void __launch_bounds__(256) distance_buckets_kernel(const float* coords, const int32_t* num_atoms, int B, int N, const __grid_constant__ Edges edges,
                                                               int n_edges, uint8_t* out, long long batch_stride, long long row) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x, square = (long long)N * N;
  if (at >= B * square) return;
  const int b = at / square, i = at % square / N, j = at % N;
  const int n = num_atoms ? num_atoms[b] : N;
  int count = 0;
  if (i < n && j < n) {
    const float *x = coords + ((long long)b * N + i) * 3, *y = coords + ((long long)b * N + j) * 3;
    const double dx = (double)x[0] - y[0], dy = (double)x[1] - y[1], dz = (double)x[2] - y[2];
    const double d2 = __dadd_rn(__dadd_rn(__dmul_rn(dx, dx), __dmul_rn(dy, dy)), __dmul_rn(dz, dz));
    for (int e = 0; e < n_edges; ++e) count += d2 >= edges.square[e];
  }
  out[b * batch_stride + i * row + j] = (uint8_t)count;
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
  MF_CHECK_ARG(table == (a->bucket_kind != MF_BUCKETS_NONE) && table == (a->buckets != nullptr), "%s: bias, buckets and bucket_kind go together", name);
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

struct BwdSpace {
  size_t delta, part, total;
  int tiles;
};
BwdSpace bwd_space(const MfDenseAttnArgs& a) {
  BwdSpace s{};
  s.tiles = dense_attn_mma_tiles(a.queries);
  s.delta = 0;
  s.part = align_up((size_t)a.batch * a.heads * a.queries * sizeof(float), 256);
  s.total = s.part + (a.bias && a.dbias ? align_up((size_t)a.batch * a.heads * s.tiles * a.num_buckets * sizeof(float), 256) : 0);
  return s;
}

}  // namespace
}  // namespace mf

extern "C" {

size_t mf_dense_attn_fwd_workspace_bytes(const MfDenseAttnArgs*) { return 0; }
size_t mf_dense_attn_bwd_workspace_bytes(const MfDenseAttnArgs* a) {
  if (!a || a->batch < 0 || a->heads < 1 || a->queries < 0 || a->num_buckets < 0) return 0;
  return mf::bwd_space(*a).total;
}

int mf_dense_attn_fwd(const MfDenseAttnArgs* a, void* stream_) {
  using namespace mf;
  const int rc = check_args("mf_dense_attn_fwd", a);
  if (rc != MF_OK) return rc;
  if (a->batch == 0 || a->queries == 0) return MF_OK;
  return dense_attn_mma_fwd(params_of(*a), a->dtype, a->head_dim, a->bucket_kind, static_cast<cudaStream_t>(stream_));
}

int mf_dense_attn_bwd(const MfDenseAttnArgs* a, void* stream_) {
  using namespace mf;
  const char* name = "mf_dense_attn_bwd";
  int rc = check_args(name, a);
  if (rc != MF_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->batch == 0) return MF_OK;
  const BwdSpace space = bwd_space(*a);
  MF_CHECK_ARG(space.total == 0 || (a->workspace && a->workspace_bytes >= space.total && aligned16(a->workspace)), "%s: %zu bytes of workspace needed, got %zu", name,
               space.total, a->workspace_bytes);
  MF_CHECK_ARG(a->queries == 0 || (a->grad_out && a->lse), "%s: grad_out and lse must not be NULL", name);
  if ((a->queries > 0 && MF_OK != (rc = check_rows(name, "grad_out", a->grad_out, a->grad_out_rows))) ||
      (a->dq && MF_OK != (rc = check_rows(name, "dq", a->dq, a->dq_rows))) || (a->dk && MF_OK != (rc = check_rows(name, "dk", a->dk, a->dk_rows))) ||
      (a->dv && MF_OK != (rc = check_rows(name, "dv", a->dv, a->dv_rows))))
    return rc;
  DenseParams p = params_of(*a);
  char* ws = static_cast<char*>(a->workspace);
  p.delta = reinterpret_cast<float*>(ws + space.delta);
  const bool table = a->bias && a->dbias;
  if (table) p.dbias_part = reinterpret_cast<float*>(ws + space.part);
  rc = dense_attn_mma_bwd(p, a->dtype, a->head_dim, a->bucket_kind, stream);
  if (rc != MF_OK || !table) return rc;
  bias_sum_kernel<<<a->heads * a->num_buckets, 128, 0, stream>>>(p.dbias_part, a->batch, a->heads, space.tiles, a->num_buckets, a->dbias, a->bias_dtype);
  MF_CHECK_LAUNCH("dense attention table gradient");
  return MF_OK;
}

int mf_distance_buckets(const float* coords, const int32_t* num_atoms, int32_t batch, int32_t tokens, const double* edges, int32_t num_edges, uint8_t* buckets,
                        int64_t batch_stride, int64_t row, void* stream) {
  using namespace mf;
  const char* name = "mf_distance_buckets";
  MF_CHECK_ARG(batch >= 0 && tokens >= 0 && tokens <= 1 << 20 && (long long)batch * tokens * tokens < (1ll << 39), "%s: sizes out of range: %d molecules of %d atoms", name, batch, tokens);
  MF_CHECK_ARG(num_edges >= 0 && num_edges <= kMaxEdges && (num_edges == 0 || edges), "%s: at most %d edges, got %d", name, kMaxEdges, num_edges);
  Edges e{};
  for (int i = 0; i < num_edges; ++i) {
    MF_CHECK_ARG(edges[i] >= 0.0 && (i == 0 || edges[i] >= edges[i - 1]), "%s: edges must ascend from 0 on", name);
    e.square[i] = edges[i] * edges[i];
  }
  if (batch == 0 || tokens == 0) return MF_OK;
  MF_CHECK_ARG(coords && buckets && row >= tokens && batch_stride >= (int64_t)(tokens - 1) * row + tokens, "%s: rows of the buckets must hold %d entries", name, tokens);
  const long long pairs = (long long)batch * tokens * tokens;
  distance_buckets_kernel<<<(unsigned)((pairs + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(coords, num_atoms, batch, tokens, e, num_edges, buckets, batch_stride,
                                                                                                       row);
  MF_CHECK_LAUNCH(name);
  return MF_OK;
}

}  // extern "C"
