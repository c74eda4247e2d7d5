// What the tcgen05 kernels of dense attention share.
#pragma once

#include "dense_attn.cuh"
#include "sm100_primitives.cuh"
#include "tensor_map.cuh"

namespace mf {

constexpr int kTcRows = 128;  // rows of a tile, queries and keys

struct DenseTcParams {
  DenseParams p;
  CUtensorMap q, k, v, grad_out;  // {head_dim, tokens, heads, batch}, boxes of 64 channels x 128 rows (forward) or 64 (backward), 128-byte swizzle
  BoundedWaits waits;
  // forward: pieces of the keys, of piece_tiles tiles each, and where they leave their rows where there are several
  int pieces = 1, piece_tiles = 0;
  float *acc = nullptr, *stat = nullptr;
};

// Instruction descriptor of kind::f16 for 16-bit operands and fp32 sums.
template <typename T>
__host__ __device__ constexpr uint32_t make_idesc_16(int m, int n, bool a_mn_major, bool b_mn_major) {
  const uint32_t d = make_idesc_bf16(m, n, a_mn_major, b_mn_major);
  return std::is_same<T, __nv_bfloat16>::value ? d : d & ~((1u << 7) | (1u << 10));
}

// A box of 64 channels, from `channel` on (a multiple of 64).
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int channel, int row, int head, int batch, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
      "r"(channel), "r"(row), "r"(head), "r"(batch), "r"((uint32_t)__cvta_generic_to_shared(bar))
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void group_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Maps of the call's operands; false where the copy engine does not take them.
bool dense_tc_maps(DenseTcParams& tc, int dtype, int head_dim, bool backward);
// Whether the call is of a kind that the 128-row kernels take, whatever its size.
bool dense_tc_takes(const DenseParams& p, int head_dim, int bucket_kind);
// The last expired wait of the forward or the backward kernels' calls (word 0) or self-test (word 1), once; synchronises.
int dense_attn_take_fwd_status(int word, int32_t* host_status, cudaStream_t stream);
int dense_attn_take_bwd_status(int word, int32_t* host_status, cudaStream_t stream);
size_t dense_tc_fwd_workspace_bytes(const DenseParams& p, int head_dim);
int dense_attn_sm100_fwd(const DenseParams& p, int dtype, int head_dim, int bucket_kind, void* workspace, cudaStream_t stream, BoundedWaits waits = {});
bool dense_tc_bwd_takes(const DenseParams& p, int head_dim, int bucket_kind, bool table_grad);
int dense_attn_sm100_bwd(const DenseTcParams& tc, int dtype, int head_dim, int bucket_kind, cudaStream_t stream);

}  // namespace mf
