// Gated feed-forward block: y = h Wo^T + bo, h = act(g) * u, [g u] = x [Wg; Wu]^T + b (T tokens, C channels, F hidden).
//
// Forward, two products: one forms g and u of 128 hidden channels side by side in tensor memory and stores h (in training g and u as
// well), one multiplies h with Wo.  Backward, four: dh = dy Wo, whose epilogue turns dh into dg = dh u act'(g) and du = dh act(g)
// where they stand (dh is never stored); dx = [dg du] [Wg; Wu]; and the weights' gradients [dg du]^T x and dy^T h.
// h, g, u, dg, du are rounded to 16 bits on their way through memory: the tensor cores take no wider operands, and g and u in 32 bits
// would double what the first product stores.  Every sum is in 32 bits.
#include "common.cuh"
#include "gemm_sm100.cuh"

namespace mf {
namespace {

using namespace gemm;

constexpr int kPairs = 74;  // clusters of two CTAs on 148 SMs
const char* const kName = "mf_gated_mlp";

// 2-D map of a row-major matrix of 16-bit elements, boxes of 64 columns.
template <typename T>
bool map16(CUtensorMap* map, const void* base, long long rows, long long cols, long long row_stride, int box_rows) {
  const long long dims[2] = {cols, rows}, strides[1] = {row_stride * 2};
  return make_tensor_map(map, base, std::is_same<T, __nv_bfloat16>::value ? MF_DTYPE_BF16 : MF_DTYPE_F16, 2, dims, strides, 64, box_rows);
}

int clusters(long long tiles) { return (int)(tiles < kPairs ? tiles : kPairs); }

template <typename T, bool kAMn, bool kBMn, int kN, Epilogue kEpi>
int launch(const Params& p, cudaStream_t stream, const char* what) {
  auto kernel = gemm_kernel<T, kAMn, kBMn, kN, kEpi>;
  constexpr int kSmem = Shape<kN, kEpi>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return cuda_error(e, what);
  const long long tiles = (long long)((p.m + 255) / 256) * ((p.n + (kEpi == kGate ? kN / 2 : kN) - 1) / (kEpi == kGate ? kN / 2 : kN)) * p.splits;
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = 2, attributes[0].val.clusterDim.y = 1, attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(2 * clusters(tiles)), config.blockDim = dim3(kThreads), config.dynamicSmemBytes = kSmem, config.stream = stream;
  config.attrs = attributes, config.numAttrs = 2;
  const cudaError_t l = cudaLaunchKernelEx(&config, kernel, p);
  return l == cudaSuccess ? MF_OK : cuda_error(l, what);
}

// ---- planes of partial sums ----------------------------------------------------------------------------------------
template <typename TOut>
__global__ void add_planes_kernel(const float* __restrict__ planes, int n, long long count, TOut* __restrict__ out) {
  wait_for_previous();
  const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (i >= count) return;
  float4 s = *reinterpret_cast<const float4*>(planes + i);
  for (int k = 1; k < n; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(planes + k * count + i);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  if constexpr (sizeof(TOut) == 4) {
    *reinterpret_cast<float4*>(out + i) = s;
  } else {
    *reinterpret_cast<uint2*>(out + i) = make_uint2(pack2<TOut>(s.x, s.y), pack2<TOut>(s.z, s.w));
  }
}

// How many pieces the tokens are cut into for a weight gradient of `tiles` tiles: the piece count with the shortest longest run of 64-token
// blocks, each plane of sums counted with what it moves.
int token_splits(long long tiles, int k_blocks, long long values) {
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 16 && (s == 1 || k_blocks / s >= 8); ++s) {
    const int per = (k_blocks + s - 1) / s;
    if ((k_blocks + per - 1) / per != s) continue;
    const double blocks = (double)((tiles * s + kPairs - 1) / kPairs) * per * 0.29, planes = s > 1 ? 8e-6 * s * (double)values / 6.5 : 0.;
    if (blocks + planes < least) least = blocks + planes, best = s;
  }
  return best;
}

struct Weight {  // gradient of an (m, n) weight over the tokens
  int m, n, splits, per_split;
};
Weight weight_plan(long long rows, int m, int n) {
  const long long tiles = (long long)((m + 255) / 256) * ((n + 255) / 256);
  const int k_blocks = (int)((rows + kBlockK - 1) / kBlockK);
  const int s = token_splits(tiles, k_blocks, (long long)m * n);
  return {m, n, s, (k_blocks + s - 1) / s};
}

size_t pieces(const MfGatedMlpArgs* a, bool backward, size_t (&at)[4]) {  // gradient of the pre-activations | planes | bias sums | their bands
  const size_t size = 2, rows = (size_t)a->rows, F = a->hidden;
  at[0] = 0;
  if (!backward || rows == 0) return 0;
  at[1] = at[0] + align_up(rows * 2 * F * size, 256);
  size_t planes = 0;
  if (a->grad_w_in) {
    const Weight w = weight_plan(a->rows, 2 * a->hidden, a->dim);
    if (w.splits > 1) planes = (size_t)w.splits * w.m * w.n * 4;
  }
  if (a->grad_w_out) {
    const Weight w = weight_plan(a->rows, a->dim_out, a->hidden);
    if (w.splits > 1 && (size_t)w.splits * w.m * w.n * 4 > planes) planes = (size_t)w.splits * w.m * w.n * 4;
  }
  at[2] = at[1] + align_up(planes, 256);
  const long long bands = (a->rows + 31) / 32;
  at[3] = at[2] + (a->grad_b_in ? align_up((size_t)bands * 2 * F * 4, 256) : 0);
  size_t sums = 0;
  if (a->grad_b_in) sums = column_sums_workspace(bands, 2 * a->hidden);
  if (a->grad_b_out && column_sums_workspace(a->rows, a->dim_out) > sums) sums = column_sums_workspace(a->rows, a->dim_out);
  return at[3] + align_up(sums, 256);
}

int check(const MfGatedMlpArgs* a) {
  MF_CHECK_ARG(a != nullptr, "%s: null argument struct", kName);
  MF_CHECK_ARG(a->dtype == MF_DTYPE_BF16 || a->dtype == MF_DTYPE_F16, "%s: only supports float16/bfloat16 inputs, got dtype code %d", kName, (int)a->dtype);
  MF_CHECK_ARG(a->grad_dtype == a->dtype || a->grad_dtype == MF_DTYPE_F32, "%s: weight gradients come in the inputs' type or in float32, got dtype code %d", kName, (int)a->grad_dtype);
  MF_CHECK_ARG(a->activation == MF_ACT_SILU || a->activation == MF_ACT_GELU_TANH, "%s: unknown activation code %d", kName, (int)a->activation);
  MF_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31) - 512, "%s: rows must lie in [0, 2^31 - 512)", kName);
  MF_CHECK_ARG(a->dim >= 8 && a->hidden >= 8 && a->dim_out >= 8 && a->dim % 8 == 0 && a->hidden % 8 == 0 && a->dim_out % 8 == 0,
               "%s: widths must be positive multiples of 8, got %d, %d, %d", kName, (int)a->dim, (int)a->hidden, (int)a->dim_out);
  MF_CHECK_ARG(a->dim <= (1 << 28) && a->hidden <= (1 << 28) && a->dim_out <= (1 << 28), "%s: widths above 2^28", kName);
  if (a->rows == 0) return MF_OK;
  MF_CHECK_ARG(a->x && a->w_in && a->w_out && a->act, "%s: null tensor", kName);
  MF_CHECK_ALIGNED(kName, a->x, a->w_in, a->w_out, a->b_in, a->b_out, a->pre, a->act, a->y, a->grad_y, a->grad_x, a->grad_w_in, a->grad_w_out,
                   a->grad_b_in, a->grad_b_out, a->workspace);
  return MF_OK;
}

Params common(const MfGatedMlpArgs* a, int m, int n, int k, const BoundedWaits& waits) {
  Params p{};
  p.m = m, p.n = n, p.k = k, p.splits = 1, p.k_blocks_per_split = (k + kBlockK - 1) / kBlockK;
  p.activation = a->activation, p.waits = waits;
  return p;
}

#define MF_MAP(call)                                                                                           \
  do {                                                                                                         \
    if (!(call)) {                                                                                             \
      set_error("%s: tensor map refused (driver code %d)", kName, last_tensor_map_result());                   \
      return MF_ERR_CUDA;                                                                                      \
    }                                                                                                          \
  } while (0)

// D (m, n) = A B^T + bias, tiles of 256 or 128 columns, whichever leaves fewer columns to the longest-running pair
template <typename T, bool kAMn, bool kBMn>
int product(Params& p, cudaStream_t stream, const char* what) {
  const long long tm = (p.m + 255) / 256, wide = (tm * ((p.n + 255) / 256) + kPairs - 1) / kPairs * 2, narrow = (tm * ((p.n + 127) / 128) + kPairs - 1) / kPairs;
  return narrow < wide ? launch<T, kAMn, kBMn, 128, kStore>(p, stream, what) : launch<T, kAMn, kBMn, 256, kStore>(p, stream, what);
}

template <typename T>
int forward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const long long M = a->rows, C = a->dim, F = a->hidden, O = a->dim_out;
  const T* w_in = static_cast<const T*>(a->w_in);
  Params p = common(a, (int)M, (int)F, (int)C, waits);
  p.bias = a->b_in, p.keep_pre = a->pre != nullptr;
  MF_MAP(map16<T>(&p.a, a->x, M, C, C, 64));
  MF_MAP(map16<T>(&p.b, w_in, F, C, C, 64));
  MF_MAP(map16<T>(&p.b2, w_in + F * C, F, C, C, 64));
  MF_MAP(map16<T>(&p.out, a->act, M, F, F, 32));
  if (a->pre) {
    MF_MAP(map16<T>(&p.pre, a->pre, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.pre2, static_cast<T*>(a->pre) + F, M, F, 2 * F, 32));
  }
  int rc = launch<T, false, false, 256, kGate>(p, stream, "gated_mlp gate product");
  if (rc != MF_OK) return rc;
  p = common(a, (int)M, (int)O, (int)F, waits);
  p.bias = a->b_out;
  MF_MAP(map16<T>(&p.a, a->act, M, F, F, 64));
  MF_MAP(map16<T>(&p.b, a->w_out, O, F, F, 64));
  MF_MAP(map16<T>(&p.out, a->y, M, O, O, 32));
  return product<T, false, false>(p, stream, "gated_mlp output product");
}

// gradient (m, n) of a weight: the sum over the tokens of left (tokens, m) x right (tokens, n)
template <typename T>
int weight_gradient(const MfGatedMlpArgs* a, const void* left, int m, const void* right, int n, void* out, float* planes, const BoundedWaits& waits,
                    cudaStream_t stream) {
  const Weight w = weight_plan(a->rows, m, n);
  Params p = common(a, m, n, (int)a->rows, waits);
  p.splits = w.splits, p.k_blocks_per_split = w.per_split;
  MF_MAP(map16<T>(&p.a, left, a->rows, m, m, 64));
  MF_MAP(map16<T>(&p.b, right, a->rows, n, n, 64));
  const bool direct = w.splits == 1;
  if (direct && a->grad_dtype != MF_DTYPE_F32) {
    MF_MAP(map16<T>(&p.out, out, m, n, n, 32));
    return launch<T, true, true, 256, kStore>(p, stream, "gated_mlp weight gradient");
  }
  const long long dims[3] = {n, m, w.splits}, strides[2] = {4ll * n, 4ll * n * m};
  MF_MAP(make_tensor_map(&p.out, direct ? out : planes, MF_DTYPE_F32, 3, dims, strides, 32, 32));
  const int rc = launch<T, true, true, 256, kStoreF32>(p, stream, "gated_mlp weight gradient");
  if (rc != MF_OK || direct) return rc;
  const long long count = (long long)m * n;
  const dim3 grid((unsigned)((count / 4 + 255) / 256));
  if (a->grad_dtype == MF_DTYPE_F32) launch_dependent(add_planes_kernel<float>, grid, dim3(256), 0, stream, planes, w.splits, count, static_cast<float*>(out));
  else launch_dependent(add_planes_kernel<T>, grid, dim3(256), 0, stream, planes, w.splits, count, static_cast<T*>(out));
  MF_CHECK_LAUNCH("add_planes_kernel");
  return MF_OK;
}

template <typename T>
int backward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const long long M = a->rows, C = a->dim, F = a->hidden, O = a->dim_out;
  size_t at[4];
  pieces(a, true, at);
  char* ws = static_cast<char*>(a->workspace);
  T* grad_pre = reinterpret_cast<T*>(ws + at[0]);
  float *planes = reinterpret_cast<float*>(ws + at[1]), *sums = reinterpret_cast<float*>(ws + at[2]), *bands = reinterpret_cast<float*>(ws + at[3]);
  int rc;
  if (a->grad_x || a->grad_w_in || a->grad_b_in) {
    Params p = common(a, (int)M, (int)F, (int)O, waits);
    p.column_sums = a->grad_b_in ? sums : nullptr;
    MF_MAP(map16<T>(&p.a, a->grad_y, M, O, O, 64));
    MF_MAP(map16<T>(&p.b, a->w_out, O, F, F, 64));
    MF_MAP(map16<T>(&p.pre, a->pre, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.pre2, static_cast<const T*>(a->pre) + F, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.out, grad_pre, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.out2, grad_pre + F, M, F, 2 * F, 32));
    if ((rc = launch<T, false, true, 256, kGateGrad>(p, stream, "gated_mlp gate gradient")) != MF_OK) return rc;
  }
  if (a->grad_x) {
    Params p = common(a, (int)M, (int)C, (int)(2 * F), waits);
    MF_MAP(map16<T>(&p.a, grad_pre, M, 2 * F, 2 * F, 64));
    MF_MAP(map16<T>(&p.b, a->w_in, 2 * F, C, C, 64));
    MF_MAP(map16<T>(&p.out, a->grad_x, M, C, C, 32));
    if ((rc = product<T, false, true>(p, stream, "gated_mlp input gradient")) != MF_OK) return rc;
  }
  if (a->grad_w_in && (rc = weight_gradient<T>(a, grad_pre, (int)(2 * F), a->x, (int)C, a->grad_w_in, planes, waits, stream)) != MF_OK) return rc;
  if (a->grad_w_out && (rc = weight_gradient<T>(a, a->grad_y, (int)O, a->act, (int)F, a->grad_w_out, planes, waits, stream)) != MF_OK) return rc;
  if (a->grad_b_in && (rc = column_sums(sums, MF_DTYPE_F32, (M + 31) / 32, (int)(2 * F), a->grad_b_in, a->grad_dtype, bands, stream)) != MF_OK) return rc;
  if (a->grad_b_out && (rc = column_sums(a->grad_y, a->dtype, M, (int)O, a->grad_b_out, a->grad_dtype, bands, stream)) != MF_OK) return rc;
  return MF_OK;
}

int run_forward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const int rc = check(a);
  if (rc != MF_OK || a->rows == 0) return rc;
  MF_CHECK_ARG(a->y, "%s: null tensor", kName);
  return a->dtype == MF_DTYPE_BF16 ? forward<__nv_bfloat16>(a, waits, stream) : forward<__half>(a, waits, stream);
}

int run_backward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const int rc = check(a);
  if (rc != MF_OK) return rc;
  if (a->rows == 0) {  // sums over no tokens
    const size_t size = a->grad_dtype == MF_DTYPE_F32 ? 4 : 2, C = a->dim, F = a->hidden, O = a->dim_out;
    void* const ptr[4] = {a->grad_w_in, a->grad_w_out, a->grad_b_in, a->grad_b_out};
    const size_t count[4] = {2 * F * C, O * F, 2 * F, O};
    for (int i = 0; i < 4; ++i)
      if (ptr[i]) {
        const cudaError_t e = cudaMemsetAsync(ptr[i], 0, count[i] * size, stream);
        if (e != cudaSuccess) return cuda_error(e, kName);
      }
    return MF_OK;
  }
  MF_CHECK_ARG(a->grad_y && a->pre, "%s: null tensor", kName);
  size_t at[4];
  const size_t need = pieces(a, true, at);
  if (need && (!a->workspace || a->workspace_bytes < need)) {
    set_error("%s: workspace too small (%zu bytes needed)", kName, need);
    return MF_ERR_WORKSPACE_TOO_SMALL;
  }
  return a->dtype == MF_DTYPE_BF16 ? backward<__nv_bfloat16>(a, waits, stream) : backward<__half>(a, waits, stream);
}

int read_status(int32_t* host_status, cudaStream_t stream, bool clear) {
  static const int32_t kNone = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(host_status, g_gemm_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbolAsync(g_gemm_status, &kNone, sizeof(int32_t), 0, cudaMemcpyHostToDevice, stream);
  if (e == cudaSuccess && clear) e = cudaStreamSynchronize(stream);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "gated_mlp status read-back");
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" size_t mf_gated_mlp_bwd_workspace_bytes(const MfGatedMlpArgs* a) {
  if (!a || a->rows < 0 || a->hidden < 1 || a->dim < 1 || a->dim_out < 1) return 0;
  size_t at[4];
  return pieces(a, true, at);
}
extern "C" int mf_gated_mlp_fwd(const MfGatedMlpArgs* a, void* stream) { return run_forward(a, BoundedWaits{}, static_cast<cudaStream_t>(stream)); }
extern "C" int mf_gated_mlp_bwd(const MfGatedMlpArgs* a, void* stream) { return run_backward(a, BoundedWaits{}, static_cast<cudaStream_t>(stream)); }
extern "C" int mf_gated_mlp_status(int32_t* host_status, void* stream) {
  MF_CHECK_ARG(host_status != nullptr, "mf_gated_mlp_status: null pointer");
  return read_status(host_status, static_cast<cudaStream_t>(stream), false);
}
extern "C" int mf_selftest_gated_mlp_give_up(const MfGatedMlpArgs* a, int32_t backward, int32_t kind, int64_t limit_cycles, int32_t* host_status,
                                             void* stream) {
  MF_CHECK_ARG(a && host_status && kind >= 0 && kind <= 3, "mf_selftest_gated_mlp_give_up: bad argument");
  MF_CHECK_ARG(limit_cycles > 0 && limit_cycles <= kWaitLimitCycles, "mf_selftest_gated_mlp_give_up: the limit must lie in (0, 2^31] clocks");
  BoundedWaits waits;
  waits.limit = limit_cycles, waits.withheld = kind;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = backward ? run_backward(a, waits, s) : run_forward(a, waits, s);
  return rc != MF_OK ? rc : read_status(host_status, s, true);
}
