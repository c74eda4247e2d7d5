// Gated feed-forward block for few tokens (one molecule, single tokens): both products stream the weights once.
//
// With at most 32 tokens every weight meets few operands: reading the weights bounds the block, 2 bytes for 2 * 32 operations at most.  The
// weights are the 16-row operand of mma.sync, the tokens its 8 columns, so that one token costs what eight do and nothing is
// padded to a 256-row tile.  A CTA owns 16 hidden channels (of gate and of up) or 16 output channels; its eight warps, and those
// of up to four CTAs of a cluster where there are few channels, share the contracted dimension, and their sums meet in shared memory,
// added in the order of warps and CTAs.  A lane reads 16 bytes of a weight row and of a token at a time: which k an operand's register
// stands for is free as long as both sides agree, so no layout of the instruction reaches memory.  29 tokens of 512 x 2048 take 11 us, two
// launches and little else (6.3 MB); one token of 4096 x 10 928 51 us, 269 MB at 5.2 TB/s.
#include "common.cuh"
#include "gated_mlp.cuh"

namespace mf {
namespace {

constexpr int kWarps = 8;
constexpr int kStep = 32;  // k of one step: 16 bytes for each of four lanes
constexpr int kBatch = 2;  // steps in flight
constexpr int kHeld = 4;   // steps whose weights a warp may hold while it waits

struct SmallParams {
  const void* x;     // (rows, k)
  const void* w;     // (n, k); kGate: (2 n, k)
  const void* bias;  // (n) or (2 n), or null
  void* out;         // (rows, n)
  void* pre;         // kGate: pre-activations (rows, 2 n) or null
  uint8_t* exponents;
  int rows, n, k;
  int activation;
  int early;  // kGate: an output product follows that loads its weights before it waits (kOutHolds)
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Plain loads: the kernel before this one may still write what they read when this one begins, and a load that is marked as read-only may
// be moved above the wait for it.
__device__ __forceinline__ uint4 load16(const void* base, size_t bytes, bool valid) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (valid) v = *reinterpret_cast<const uint4*>(static_cast<const char*>(base) + bytes);
  return v;
}
// weights are read once: past L1
__device__ __forceinline__ uint4 stream16(const void* base, size_t bytes, bool valid) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (valid)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(static_cast<const char*>(base) + bytes));
  return v;
}

// the same from L2: what an earlier kernel wrote
__device__ __forceinline__ uint4 stream16_l2(const void* base, size_t bytes, bool valid) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (valid)
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(static_cast<const char*>(base) + bytes)
                 : "memory");
  return v;
}

// kTiles: of eight tokens.  kOutHolds: the output product where a warp has at most kHeld steps; it loads their weights before it waits for
// the hidden values (us, without | with: 512 x 2048, one token 5.4 | 5.0, sixteen 9.7 | 7.7, 32 13.0 | 11.1; 1024 x 4096, one 12.6 | 11.5, sixteen
// 15.2 | 14.3; with up to eight steps 2048 x 8192 24.0 | 26.7).
enum Product { kGate, kOut, kOutHolds };
template <typename T, int kTiles, Product kProduct>
__global__ void __launch_bounds__(kWarps * 32) small_kernel(const SmallParams p) {
  constexpr bool kGates = kProduct == kGate;
  constexpr int kSides = kGates ? 2 : 1, kRows = 16 * kSides, kTokens = 8 * kTiles;
  __shared__ float part[kWarps][kRows][kTokens + 1];
  __shared__ float sums[kRows][kTokens + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int n0 = (int)(blockIdx.x / ranks) * 16;
  const int steps = (p.k + kStep - 1) / kStep, slices = kWarps * (int)ranks, slice = (int)rank * kWarps + warp;
  const int s0 = (int)((long long)steps * slice / slices), s1 = (int)((long long)steps * (slice + 1) / slices);

  size_t row[kSides][2];  // byte offsets of this lane's two weight rows
  bool ok[2] = {n0 + g < p.n, n0 + g + 8 < p.n};
#pragma unroll
  for (int side = 0; side < kSides; ++side)
#pragma unroll
    for (int r = 0; r < 2; ++r) row[side][r] = ((size_t)side * p.n + n0 + g + 8 * r) * p.k * 2;
  // The gate product reads no value before the kernels before it have ended; a short slice of its weights may already move to L2 (29 tokens,
  // 512 x 2048: a microsecond of 14; long slices are slower for it, 57 -> 64 us for one token of 4096 x 10 928).  Where it lets the output product
  // begin only then, all that came before the gate product has ended and been written when that one begins, so its weights are there.
  if (!kGates || !p.early) launch_dependents();
  if (kGates && s1 - s0 <= 4 && s0 + t < s1)  // (64 bytes of a row a step: one lane in four asks for each)
#pragma unroll
    for (int side = 0; side < kSides; ++side)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (ok[r]) asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(p.w) + row[side][r] + (size_t)(s0 + t) * (2 * kStep)));

  float acc[kSides][kTiles][4] = {};
  auto add = [&](const uint4 (&w)[kSides][2], const uint4 (&x)[kTiles]) {
#pragma unroll
    for (int side = 0; side < kSides; ++side) {
      const uint4 lo = w[side][0], hi = w[side][1];
      const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        mma<T>(acc[side][n], a0, x[n].x, x[n].y);
        mma<T>(acc[side][n], a1, x[n].z, x[n].w);
      }
    }
  };
  if constexpr (kProduct == kOutHolds) {
    uint4 w[kHeld][kSides][2];
    auto valid = [&](int b) { return s0 + b < s1 && (s0 + b) * kStep + 8 * t < p.k; };
#pragma unroll
    for (int b = 0; b < kHeld; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r) w[b][0][r] = stream16_l2(p.w, row[0][r] + ((size_t)(s0 + b) * kStep + 8 * t) * 2, valid(b) && ok[r]);
    wait_for_previous();
#pragma unroll
    for (int i = 0; i < kHeld; i += kBatch) {
      uint4 x[kBatch][kTiles];
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          x[b][n] = load16(p.x, ((size_t)(8 * n + g) * p.k + (s0 + i + b) * kStep + 8 * t) * 2, valid(i + b) && 8 * n + g < p.rows);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) add(w[i + b], x[b]);
    }
  } else {
    wait_for_previous();
    if (kGates && p.early) launch_dependents();
    for (int s = s0; s < s1; s += kBatch) {
      uint4 w[kBatch][kSides][2], x[kBatch][kTiles];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int k = (s + b) * kStep + 8 * t;
        const bool in = s + b < s1 && k < p.k;
#pragma unroll
        for (int side = 0; side < kSides; ++side)
#pragma unroll
          for (int r = 0; r < 2; ++r) w[b][side][r] = stream16(p.w, row[side][r] + (size_t)k * 2, in && ok[r]);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) x[b][n] = load16(p.x, ((size_t)(8 * n + g) * p.k + k) * 2, in && 8 * n + g < p.rows);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) add(w[b], x[b]);
    }
  }
#pragma unroll
  for (int side = 0; side < kSides; ++side)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][16 * side + g + 8 * (i >> 1)][8 * n + 2 * t + (i & 1)] = acc[side][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kTokens; i += kWarps * 32) {
    const int r = i / kTokens, c = i % kTokens;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += part[w][r][c];
    sums[r][c] = s;
  }
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();

  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&sums[0][0]);
  auto total = [&](int r, int c) {
    if (ranks == 1) return sums[r][c];
    float s = 0.f;
    for (uint32_t q = 0; q < ranks; ++q) {
      uint32_t at;
      float v;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + 4u * (uint32_t)(r * (kTokens + 1) + c)), "r"(q));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
      s += v;
    }
    return s;
  };
  const T* bias = static_cast<const T*>(p.bias);
  const bool biased = bias != nullptr;
  // the CTAs of a cluster store every ranks-th token; sixteen lanes hold a token's channels
  for (int i = threadIdx.x; i < 16 * kTokens; i += kWarps * 32) {
    const int r = i & 15, c = i >> 4, n = n0 + r;
    if (c >= p.rows || c % ranks != rank) continue;
    float a = total(r, c);
    if (biased && n < p.n) a += to_f32(bias[n]);
    if constexpr (kGates) {
      float u = total(16 + r, c);
      if (biased && n < p.n) u += to_f32(bias[p.n + n]);
      if (p.pre) {
        const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
        PreGroup<T> of_gate, of_up;
        of_gate.add(a, a), of_up.add(u, u);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) of_gate.exchange(lanes, o), of_up.exchange(lanes, o);
        const uint32_t eg = of_gate.code(), eu = of_up.code();
        if (n < p.n) {
          uint16_t* pre = static_cast<uint16_t*>(p.pre) + (size_t)c * 2 * p.n + n;
          pre[0] = (uint16_t)PreForm<T>(eg, false).pack(make_float2(a, 0.f)), pre[p.n] = (uint16_t)PreForm<T>(eu, false).pack(make_float2(u, 0.f));
        }
        if (r == 0) {
          uint8_t* to = p.exponents + ((size_t)(n0 >> 6) * p.rows + c) * 8 + ((n0 >> 4) & 3);
          to[0] = (uint8_t)eg, to[4] = (uint8_t)eu;
        }
      }
      const float2 f = p.activation == MF_ACT_SILU ? activation2<MF_ACT_SILU>(make_float2(a, a)) : activation2<MF_ACT_GELU_TANH>(make_float2(a, a));
      a = f.x * u;
    }
    if (n < p.n) static_cast<T*>(p.out)[(size_t)c * p.n + n] = from_f32<T>(a);
  }
  if (ranks > 1) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");  // the sums stay until all have read
}

int ranks_of(int n, int k) {
  const int tiles = (n + 15) / 16, steps = (k + kStep - 1) / kStep;
  // Enough CTAs for two on every SM, while a warp keeps two steps at least.  Sums over a cluster cost more than idle SMs beyond that: 16 tokens,
  // 1024 x 4096: clusters of 4 15 us, of 8 23 us; one token, 4096 x 10 928: two CTAs an SM 53 us, four 55, eight 82.
  int ranks = 1;
  while (ranks < 4 && tiles * ranks < 2 * 148 && steps / (2 * ranks * kWarps) >= 2) ranks *= 2;
  return ranks;
}

template <typename T, int kTiles, Product kProduct>
int launch(const SmallParams& p, cudaStream_t stream, const char* what) {
  const int tiles = (p.n + 15) / 16, ranks = ranks_of(p.n, p.k);
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = ranks, attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(tiles * ranks)), config.blockDim = dim3(kWarps * 32), config.stream = stream;
  config.attrs = attributes, config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, small_kernel<T, kTiles, kProduct>, p);
  return e == cudaSuccess ? MF_OK : cuda_error(e, what);
}

template <typename T, Product kProduct>
int launch_tokens(const SmallParams& p, cudaStream_t stream, const char* what) {
  return p.rows <= 8 ? launch<T, 1, kProduct>(p, stream, what) : p.rows <= 16 ? launch<T, 2, kProduct>(p, stream, what) : launch<T, 4, kProduct>(p, stream, what);
}

template <typename T>
int forward(const MfGatedMlpArgs* a, cudaStream_t stream) {
  const int rows = (int)a->rows;
  uint8_t* exponents = a->pre ? static_cast<uint8_t*>(a->pre) + gated_mlp_pre_values(rows, a->hidden) : nullptr;
  const int early = (a->hidden + kStep - 1) / kStep <= kHeld * kWarps * ranks_of(a->dim_out, a->hidden);
  const int rc = launch_tokens<T, kGate>({a->x, a->w_in, a->b_in, a->act, a->pre, exponents, rows, a->hidden, a->dim, a->activation, early}, stream, "gated_mlp gate product");
  if (rc != MF_OK) return rc;
  const SmallParams out = {a->act, a->w_out, a->b_out, a->y, nullptr, nullptr, rows, a->dim_out, a->hidden, 0, 0};
  const char* what = "gated_mlp output product";
  return early ? launch_tokens<T, kOutHolds>(out, stream, what) : launch_tokens<T, kOut>(out, stream, what);
}

}  // namespace

int gated_mlp_small_forward(const MfGatedMlpArgs* a, cudaStream_t stream) {
  return a->dtype == MF_DTYPE_BF16 ? forward<__nv_bfloat16>(a, stream) : forward<__half>(a, stream);
}

}  // namespace mf
