// What the kernels of dense attention share: the call's operands, which keys a query sees, and the learned bias by buckets.
#pragma once

#include <atomic>

#include "common.cuh"
#include "sparse_attn_mma.cuh"

namespace mf {

constexpr float kDenseLog2e = 1.4426950408889634f;
constexpr float kDenseLn2 = 0.6931471805599453f;
constexpr float kDenseHidden = -1e30f;  // entries of the table below this hide their pairs
constexpr int kMaxBuckets = 128;
constexpr int kTableEntries = 256;  // one for every byte that may stand among the buckets

struct DenseRows {
  long long batch, head, token;
  __host__ __device__ __forceinline__ long long at(int b, int h, long long n) const { return b * batch + h * head + n * token; }
};

struct DenseParams {
  const void *q, *k, *v, *grad_out;
  void *out, *dq, *dk, *dv;
  DenseRows q_rows, k_rows, v_rows, out_rows, go_rows, dq_rows, dk_rows, dv_rows;
  const int32_t *num_queries, *num_keys;
  const uint8_t* key_mask;
  long long key_mask_batch;
  const void* bias;
  int bias_dtype, num_buckets, reach;
  const uint8_t* buckets;
  long long bucket_batch, bucket_row;
  float* lse;    // per query in units of log2; +inf where a query sees nothing
  float* delta;  // sum over the channels of grad_out * out, backward
  float* dbias_part;  // [batch * heads * query tiles][num_buckets]
  int B, H, K, M, N;  // batch, heads, key heads, queries, keys (padded)
  int causal;
  float scale;
};

// Adds four values to a lane's column of sums, in order; the sums are read together, so that a value does not wait for the one before it to be
// written (a chain of 40 clocks each): where two go to one sum, the later store holds both.
__device__ __forceinline__ void add_four(float* column, const int (&at)[4], const float (&d)[4]) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = column[at[i] * 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < i; ++j) v[i] += at[j] == at[i] ? d[j] : 0.f;
    column[at[i] * 32] = v[i] += d[i];
  }
}

struct DenseLengths {
  int nq, nk, shift;  // shift: where the first query stands among the keys
};
__device__ __forceinline__ DenseLengths dense_lengths(const DenseParams& p, int b) {
  DenseLengths n;
  n.nq = p.num_queries ? max(0, min(p.num_queries[b], p.M)) : p.M;
  n.nk = p.num_keys ? max(0, min(p.num_keys[b], p.N)) : p.N;
  n.shift = n.nk - n.nq;
  return n;
}
// keys that query i sees, as far as lengths and order say: [0, this)
__device__ __forceinline__ int dense_limit(const DenseParams& p, const DenseLengths& n, int i) {
  if (i >= n.nq) return 0;
  return p.causal ? max(0, min(n.nk, i + n.shift + 1)) : n.nk;
}
// queries that see key j: [this, nq)
__device__ __forceinline__ int dense_first(const DenseParams& p, const DenseLengths& n, int j) {
  return p.causal ? max(0, j - n.shift) : 0;
}

// Column `head` of the table in units of log2; buckets beyond the table have no bias.
__device__ __forceinline__ float dense_bias_entry(const DenseParams& p, int bucket, int head) {
  if (bucket >= p.num_buckets) return 0.f;
  const long long at = (long long)bucket * p.H + head;
  const float v = p.bias_dtype == MF_DTYPE_F32    ? static_cast<const float*>(p.bias)[at]
                  : p.bias_dtype == MF_DTYPE_BF16 ? to_f32(static_cast<const __nv_bfloat16*>(p.bias)[at])
                                                  : to_f32(static_cast<const __half*>(p.bias)[at]);
  return v < kDenseHidden ? -INFINITY : v * kDenseLog2e;
}
__device__ __forceinline__ int dense_offset_bucket(const DenseParams& p, int offset) {
  return p.buckets[max(-p.reach, min(p.reach, offset)) + p.reach];
}

// Eight bytes from `at` on, of which the first `n` are there: words that hold one of them are read, no others.
__device__ __forceinline__ uint2 eight_bytes(const uint8_t* at, int n) {
  const int skip = (int)(reinterpret_cast<uintptr_t>(at) & 3);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(at - skip);
  n = n > 8 ? 8 : n;
  const uint32_t a = n > 0 ? w[0] : 0u, b = skip + n > 4 ? w[1] : 0u, c = skip + n > 8 ? w[2] : 0u;
  return make_uint2(__funnelshift_r(a, b, 8 * skip), __funnelshift_r(b, c, 8 * skip));
}

// The first `bytes` of 16, zeros behind them; no others are read.
__device__ __forceinline__ void cp_async_part16(uint32_t smem_addr, const void* gptr, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr), "l"(gptr), "r"(bytes) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_bf16(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float dense_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Lets a kernel have `bytes` of dynamic shared memory, one value for all its calls: asked for once on a device (it takes a microsecond).
template <auto kernel>
cudaError_t allow_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess || (device < 64 && (done.load(std::memory_order_relaxed) >> device & 1))) return err;
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
  return err;
}

// dense_attn_mma.cu: any call
int dense_attn_mma_fwd(const DenseParams& p, int dtype, int head_dim, int bucket_kind, cudaStream_t stream);
int dense_attn_mma_bwd(const DenseParams& p, int dtype, int head_dim, int bucket_kind, cudaStream_t stream);
int dense_attn_mma_slots(const DenseParams& p, int head_dim);  // partial sums of the table's gradient for each head
// dense_attn_small.cu: at most 32 queries and keys
bool dense_attn_small_applies(const DenseParams& p, bool backward);
int dense_attn_small_slots(const DenseParams& p, int head_dim, int bucket_kind);  // partial sums of the table's gradient for each head
int dense_attn_small(const DenseParams& p, int dtype, int head_dim, int bucket_kind, bool backward, cudaStream_t stream);
// dense_attn_split.cu: forward, few queries
bool dense_attn_split_applies(const DenseParams& p, int head_dim);
size_t dense_attn_split_workspace_bytes(const DenseParams& p, int head_dim);
// Joins pieces of the keys: acc [entry * key head][tile of 16 rows][piece][16][D] in units of exp2(-top), stat the same without D: top, total.  A row is query * group +
// head of the group; a total of zero stands for a piece that wrote no row.  Where all logits are no numbers top is minus infinity and total none.
int dense_attn_join(const DenseParams& p, int dtype, int head_dim, int pieces, float* acc, float* stat, cudaStream_t stream);
size_t dense_attn_join_bytes(const DenseParams& p, int head_dim, int pieces);
int dense_attn_split(const DenseParams& p, int dtype, int head_dim, int bucket_kind, void* workspace, cudaStream_t stream);

}  // namespace mf
