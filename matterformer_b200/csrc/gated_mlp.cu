// Gated feed-forward block: y = h Wo^T + bo, h = act(g) * u, [g u] = x [Wg; Wu]^T + b (T tokens, C channels, F hidden).
//
// Forward, two products: one forms g and u of 128 hidden channels side by side in tensor memory and stores h (in training g and u as
// well), one multiplies h with Wo.  Backward, four: dh = dy Wo, whose epilogue turns dh into dg = dh u act'(g) and du = dh act(g)
// where they stand (dh is never stored); dx = [dg du] [Wg; Wu]; and the weights' gradients [dg du]^T x and dy^T h.
// h, dg and du are rounded to the block's type on their way through memory: the tensor cores take no wider operands.  g and u are kept
// in 16 bits of a form of their own (gated_mlp.cuh), since 32 would double what the first product stores.  Every sum is in 32 bits.
// 29 696 tokens x 512 x 2048, forward and all gradients, a pass among others on several cards: 571-611 us, 0.92-0.98 PFLOP/s (cuBLAS sustains
// 1.39 in one long product, bursts at 1.64; linear layers and element-wise operations in bf16 take 1360-1410).  Launch by launch, at 1.46-1.68
// GHz: projections 116, output 52, gate gradient 104 (495 MB, 4.8 TB/s; the tensor pipe at 37 %), gradients 203 (94 %).  8192 x 2048 x
// 5464: 1404-1474 us, 1.12-1.18 PFLOP/s.
#include <mutex>

#include "common.cuh"
#include "gemm_sm100.cuh"

namespace mf {
namespace {

using namespace gemm;

constexpr int kPairs = 74;  // clusters of two CTAs on 148 SMs
const char* const kName = "mf_gated_mlp";

// 2-D map of a row-major matrix of 16-bit elements.
template <typename T>
bool map16(CUtensorMap* map, const void* base, long long rows, long long cols, long long row_stride, int box_rows, int box_cols = 64) {
  const long long dims[2] = {cols, rows}, strides[1] = {row_stride * 2};
  return make_tensor_map(map, base, std::is_same<T, __nv_bfloat16>::value ? MF_DTYPE_BF16 : MF_DTYPE_F16, 2, dims, strides, box_cols, box_rows);
}

template <typename T, bool kAMn, bool kBMn, Epilogue kEpi, int kAct>
int launch_kernel(const Params& p, int pairs, cudaStream_t stream, const char* what) {
  auto kernel = gemm_kernel<T, kAMn, kBMn, kEpi, kAct>;
  constexpr int kSmem = Shape<kEpi>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return cuda_error(e, what);
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = 2, attributes[0].val.clusterDim.y = 1, attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(2 * pairs), config.blockDim = dim3(kThreads), config.dynamicSmemBytes = kSmem, config.stream = stream;
  config.attrs = attributes, config.numAttrs = 2;
  const cudaError_t l = cudaLaunchKernelEx(&config, kernel, p);
  return l == cudaSuccess ? MF_OK : cuda_error(l, what);
}

#define MF_MAP(call)                                                                                           \
  do {                                                                                                         \
    if (!(call)) {                                                                                             \
      set_error("%s: tensor map refused (driver code %d)", kName, last_tensor_map_result());                   \
      return MF_ERR_CUDA;                                                                                      \
    }                                                                                                          \
  } while (0)

int tiles_of(long long rows, long long cols, int width) { return (int)(((rows + kTile - 1) / kTile) * ((cols + width - 1) / width)); }

// Tiles of full width in whole rounds of the pairs; a last round that would leave at least half (three quarters) of them without work is
// cut into tiles of half (a quarter of) the width.  29 696 x 512 over 2048: 232 tiles are 3.1 rounds.
template <Epilogue kEpi>
void cut_tiles(Params& p) {
  const int tiles = tiles_of(p.one.m, p.one.n, projects(kEpi) ? kTile / 2 : kTile), rest = tiles % kPairs;
  p.cut = rest == 0 || 2 * rest > kPairs ? 1 : projects(kEpi) || 4 * rest > kPairs ? 2 : 4;
  p.whole = p.cut == 1 ? tiles : tiles - rest;
  p.tiles = p.whole + (tiles - p.whole) * p.cut;
  p.slices = 1;
}

template <typename T, bool kAMn, bool kBMn, Epilogue kEpi>
int launch(Params& p, int activation, cudaStream_t stream, const char* what) {
  const long long items = (long long)p.tiles * p.slices;
  const int pairs = (int)(items < kPairs ? items : kPairs);
  if constexpr (stores(kEpi)) return launch_kernel<T, kAMn, kBMn, kEpi, 0>(p, pairs, stream, what);
  else
    return activation == MF_ACT_SILU ? launch_kernel<T, kAMn, kBMn, kEpi, MF_ACT_SILU>(p, pairs, stream, what)
                                     : launch_kernel<T, kAMn, kBMn, kEpi, MF_ACT_GELU_TANH>(p, pairs, stream, what);
}

// ---- few tiles over a long dimension -------------------------------------------------------------------------------
// The output product of some hundred tokens: a few tiles for 74 pairs, each over all hidden channels.  Cut into narrower tiles they would
// still leave pairs idle and give the others less of the weights at a time; cut along the hidden channels, every pair reads a share of the
// weights at full width, and a second launch adds the planes and the bias.  33 tokens, 1024 x 4096: 27 -> 20 us, 2048 x 8192: 47 -> 32,
// 4096 x 10 928: 83 -> 68.  Estimated in clocks: a block of 64 channels takes 650, 250, 220 at 256, 128, 64 columns (eight stages for the
// latter two), the second launch 4500 and a clock for every 2500 bytes of planes written and read; with 560, 300, 250 and 6000 some sizes
// went whole that gain by slices: 64 tokens, 512 x 2048 15.4 -> 13.2, 128 tokens, 1024 x 2736 18.9 -> 16.0.
struct Slices {
  int cut, slices;
};
Slices slices_of(long long m, long long n, long long k) {
  const int tiles = tiles_of(m, n, kTile), k_blocks = (int)((k + kBlockK - 1) / kBlockK);
  Slices best = {0, 1};
  if (tiles > kPairs / 2) return best;
  const double clocks[5] = {0, 650, 250, 0, 220};
  const int cut = 4 * tiles <= kPairs ? 4 : 2;
  double least = (double)k_blocks * clocks[cut];
  for (int c = 1; c <= 2; c *= 2)
    for (int s = 2; tiles * c * s <= kPairs && 2 * s <= k_blocks; ++s) {
      const int per = (k_blocks + s - 1) / s;
      if ((k_blocks + per - 1) / per != s) continue;
      const double t = per * clocks[c] + 4500. + 8. * (double)m * n * s / 2500.;
      if (t < least) least = t, best = {c, s};
    }
  return best;
}
size_t slice_bytes(long long m, long long n, long long k) {
  const Slices s = slices_of(m, n, k);
  return s.slices > 1 ? (size_t)s.slices * m * n * 4 : 0;
}

template <typename T>
__global__ void __launch_bounds__(256) add_slices_kernel(const float* planes, int slices, long long values, int n, const T* bias, T* out) {
  wait_for_previous();
  const long long i = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (i >= values) return;
  float4 s = *reinterpret_cast<const float4*>(planes + i);
#pragma unroll 4
  for (int k = 1; k < slices; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(planes + k * values + i);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  if (bias) {
    const uint2 w = *reinterpret_cast<const uint2*>(bias + i % n);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    s.x += a.x, s.y += a.y, s.z += b.x, s.w += b.y;
  }
  *reinterpret_cast<uint2*>(out + i) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

// out (m, n) = A B^T + bias, in slices where that pays and `planes` is given.
template <typename T, bool kBMn>
int store_product(Params& p, const T* bias, T* out, float* planes, cudaStream_t stream, const char* what) {
  const long long m = p.one.m, n = p.one.n;
  cut_tiles<kStore>(p);
  const Slices s = planes ? slices_of(m, n, p.k) : Slices{0, 1};
  if (s.slices > 1) {
    p.cut = s.cut, p.whole = 0, p.tiles = tiles_of(m, n, kTile) * s.cut, p.slices = s.slices;
    const long long dims[3] = {n, m, s.slices}, strides[2] = {4 * n, 4 * n * m};
    MF_MAP(make_tensor_map(&p.pre, planes, MF_DTYPE_F32, 3, dims, strides, 32, 32));
  } else {
    p.bias = bias;
  }
  MF_MAP(map16<T>(&p.one.out, out, m, n, n, 32));
  const int rc = p.whole == 0 && p.cut > 1 ? launch<T, false, kBMn, kStoreNarrow>(p, 0, stream, what) : launch<T, false, kBMn, kStore>(p, 0, stream, what);
  if (rc != MF_OK || s.slices == 1) return rc;
  launch_dependent(add_slices_kernel<T>, dim3((unsigned)((m * n / 4 + 255) / 256)), dim3(256), 0, stream, planes, s.slices, m * n, (int)n, bias, out);
  MF_CHECK_LAUNCH("add_slices_kernel");
  return MF_OK;
}

// ---- gradients of the weights and of the input ---------------------------------------------------------------------
// The weights' are sums over the tokens, of [dg du] x and of dy h, the input's is [dg du] W: one launch for the tiles of all three.  Each
// pair of CTAs takes tiles of the weights in turn, which are long; those that have none in the last round take tiles of the input's
// meanwhile, from the first token on as the weights' tiles do, so that [dg du] comes from memory once for both; the rest goes round
// all pairs.  Where the weights have few tiles and many tokens, they are cut into pieces of the tokens, each with a plane of partial sums of
// its own, which add_planes_kernel adds in order.  29 696 tokens x 512 x 2048: 213 us, in launches of their own 117 + 150 + 11.
// The plan goes by the sizes alone, so that one gradient's bits do not depend on which others are wanted.
struct Plan {
  int k_blocks, tiles1, tiles, pieces, per;  // of the weights
  int first, wanted;                         // of the wanted ones
};
// Rounds of the weights' pieces and of `input` tiles of `input_blocks` blocks behind and beside them: how many a pair without a piece in the
// last round does ahead, and the longest a pair works, in blocks.
struct Rounds {
  int pairs, ahead, tiles_ahead;
  double longest;
};
Rounds rounds_of(int pieces, int blocks, int input, int input_blocks) {
  Rounds r;
  r.pairs = pieces + 4 * input < kPairs ? pieces + 4 * input : kPairs;
  const int full = pieces / r.pairs, last = pieces % r.pairs, others = r.pairs - last;
  r.ahead = last && input_blocks ? blocks / input_blocks : 0;
  r.tiles_ahead = (long long)r.ahead * others < input ? r.ahead * others : input;
  const int rest = input - r.tiles_ahead, tail = rest % r.pairs;
  const double behind = (double)(rest / r.pairs) * input_blocks + (tail == 0 ? 0. : 4 * tail <= r.pairs ? 0.4 : 2 * tail <= r.pairs ? 0.55 : 1.) * input_blocks;
  const double busy = (double)(full + (last > 0)) * blocks, free = (double)full * blocks + (double)((r.tiles_ahead + others - 1) / others) * input_blocks;
  r.longest = (busy > free ? busy : free) + behind;
  return r;
}
int input_blocks(const MfGatedMlpArgs* a) { return (2 * a->hidden + kBlockK - 1) / kBlockK; }
Plan plan_of(const MfGatedMlpArgs* a) {
  Plan w;
  w.k_blocks = (int)((a->rows + kBlockK - 1) / kBlockK);
  w.tiles1 = tiles_of(2ll * a->hidden, a->dim, kTile);
  w.tiles = w.tiles1 + tiles_of(a->dim_out, a->hidden, kTile);
  const int input = tiles_of(a->rows, a->dim, kTile);
  w.pieces = 1, w.per = w.k_blocks;
  double least = 1e30;
  for (int s = 1; s <= 16 && s <= w.k_blocks; ++s) {
    const int per = (w.k_blocks + s - 1) / s;
    if ((w.k_blocks + per - 1) / per != s) continue;  // a piece would be empty
    // a plane's way to memory and back takes a third of the 0.3 us of a block
    const double blocks = rounds_of(w.tiles * s, per, input, input_blocks(a)).longest + (s > 1 ? 0.33 * w.tiles * s : 0.);
    if (blocks < least) least = blocks, w.pieces = s, w.per = per;
  }
  w.first = a->grad_w_in ? 0 : w.tiles1;
  w.wanted = (a->grad_w_out ? w.tiles : w.tiles1) - w.first;
  return w;
}
size_t plane_bytes(const Plan& w) { return w.pieces > 1 ? (size_t)w.wanted * w.pieces * kTile * kTile * 4 : 0; }

template <typename T, typename TOut>
__global__ void __launch_bounds__(256) add_planes_kernel(const float* planes, Plan w, TOut* out1, int m1, int n1, TOut* out2, int m2, int n2) {
  wait_for_previous();
  const int tile = w.first + blockIdx.x;
  const bool second = tile >= w.tiles1;
  const int m = second ? m2 : m1, n = second ? n2 : n1;
  TOut* out = second ? out2 : out1;
  int tm, tn;
  tile_at(second ? tile - w.tiles1 : tile, (m + kTile - 1) / kTile, (n + kTile - 1) / kTile, tm, tn);
  const int row = blockIdx.y * 4 + (threadIdx.x >> 6), col = 4 * (threadIdx.x & 63);
  if (tm * kTile + row >= m || tn * kTile + col >= n) return;
  const float* from = planes + ((size_t)blockIdx.x * kTile + row) * kTile + col;
  const size_t stride = (size_t)w.wanted * kTile * kTile;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int q = 0; q < w.pieces; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(from + q * stride);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  TOut* to = out + (size_t)(tm * kTile + row) * n + tn * kTile + col;
  if constexpr (sizeof(TOut) == 4) *reinterpret_cast<float4*>(to) = s;
  else *reinterpret_cast<uint2*>(to) = make_uint2(pack2<TOut>(s.x, s.y), pack2<TOut>(s.z, s.w));
}

bool forms_pre_gradient(const MfGatedMlpArgs* a) { return a->grad_x || a->grad_w_in || a->grad_b_in; }

// The backward pass's workspace: gradient of the pre-activations | planes | bias sums | their bands
size_t pieces(const MfGatedMlpArgs* a, size_t (&at)[4]) {
  const size_t size = 2, rows = (size_t)a->rows, F = a->hidden;
  at[0] = at[1] = at[2] = at[3] = 0;
  if (rows == 0) return 0;
  at[1] = at[0] + (forms_pre_gradient(a) ? align_up(rows * 2 * F * size, 256) : 0);
  const size_t planes = a->grad_w_in || a->grad_w_out ? plane_bytes(plan_of(a)) : 0;
  at[2] = at[1] + align_up(planes, 256);
  at[3] = at[2] + (a->grad_b_in ? align_up((size_t)((a->rows + 31) / 32) * 2 * F * 4, 256) : 0);
  return at[3] + align_up((size_t)kBands * ((a->grad_b_in ? 2 * F : 0) + (a->grad_b_out ? (size_t)a->dim_out : 0)) * 4, 256);
}

// ---- gradients of the biases ---------------------------------------------------------------------------------------
// The bands' sums come from the idle warps of the launch above, where weights are wanted, else from a launch of their own.
template <typename T>
__global__ void __launch_bounds__(64) bias_bands_kernel(BiasSums b) {
  wait_for_previous();
  bias_band<T>(b, 2 * blockIdx.x + (threadIdx.x >> 5), threadIdx.x & 31);
}
// 32 columns a block; thread (x, y) adds the bands y, y + 8, ..., then the eight sums are added in order.
template <typename TOut>
__global__ void __launch_bounds__(256) add_bias_bands_kernel(BiasSums b, TOut* out_in, TOut* out_out) {
  __shared__ float red[8][32];
  wait_for_previous();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, n = b.n_in + b.n_out, c = blockIdx.x * 32 + x;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int k = y; k < kBands; k += 8) s += b.part[(size_t)k * n + c];
  }
  red[y][x] = s;
  __syncthreads();
  if (y == 0 && c < n) {
    for (int k = 1; k < 8; ++k) s += red[k][x];
    if (c < b.n_in) out_in[c] = from_f32<TOut>(s);
    else out_out[c - b.n_in] = from_f32<TOut>(s);
  }
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

Params common(long long m, long long n, long long k, const BoundedWaits& waits) {
  Params p{};
  p.one.m = (int)m, p.one.n = (int)n, p.k = (int)k, p.waits = waits;
  return p;
}

uint2* exponents_of(const MfGatedMlpArgs* a) { return reinterpret_cast<uint2*>(static_cast<char*>(a->pre) + gated_mlp_pre_values(a->rows, a->hidden)); }

template <typename T>
int forward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const long long M = a->rows, C = a->dim, F = a->hidden, O = a->dim_out;
  const T* w_in = static_cast<const T*>(a->w_in);
  Params p = common(M, F, C, waits);
  p.bias = a->b_in;
  MF_MAP(map16<T>(&p.one.a, a->x, M, C, C, 64));
  MF_MAP(map16<T>(&p.one.b, w_in, F, C, C, 64));
  MF_MAP(map16<T>(&p.b2, w_in + F * C, F, C, C, 64));
  MF_MAP(map16<T>(&p.one.out, a->act, M, F, F, 32));
  if (a->pre) {
    p.exponents = exponents_of(a);
    MF_MAP(map16<T>(&p.pre, a->pre, M, F, 2 * F, 32, 32));
    MF_MAP(map16<T>(&p.pre2, static_cast<T*>(a->pre) + F, M, F, 2 * F, 32, 32));
  }
  cut_tiles<kGate>(p);
  int rc = a->pre ? launch<T, false, false, kGateKeep>(p, a->activation, stream, "gated_mlp gate product")
                  : launch<T, false, false, kGate>(p, a->activation, stream, "gated_mlp gate product");
  if (rc != MF_OK) return rc;
  p = common(M, O, F, waits);
  MF_MAP(map16<T>(&p.one.a, a->act, M, F, F, 64));
  MF_MAP(map16<T>(&p.one.b, a->w_out, O, F, F, 64));
  float* planes = a->workspace && a->workspace_bytes >= slice_bytes(M, O, F) ? static_cast<float*>(a->workspace) : nullptr;
  return store_product<T, false>(p, static_cast<const T*>(a->b_out), static_cast<T*>(a->y), planes, stream, "gated_mlp output product");
}

// One of the two weight gradients: the sum over the tokens of left (tokens, m) x right (tokens, n).
template <typename T>
bool weight_problem(Problem& q, const MfGatedMlpArgs* a, const void* left, long long m, const void* right, long long n, void* out) {
  const long long dims[2] = {n, m}, strides[1] = {4 * n};
  q.m = (int)m, q.n = (int)n;
  return map16<T>(&q.a, left, a->rows, m, m, 64) && map16<T>(&q.b, right, a->rows, n, n, 64) &&
         (a->grad_dtype == MF_DTYPE_F32 ? make_tensor_map(&q.out, out, MF_DTYPE_F32, 2, dims, strides, 32, 32) : map16<T>(&q.out, out, m, n, n, 32));
}

template <typename T>
int gradients(const MfGatedMlpArgs* a, const void* grad_pre, float* planes, const BiasSums& bias_sums, const BoundedWaits& waits, cudaStream_t stream) {
  const int C = a->dim, F = a->hidden, O = a->dim_out;
  const Plan w = plan_of(a);
  Params p{};
  p.k = (int)a->rows, p.k_input = 2 * F, p.waits = waits, p.wide_out = a->grad_dtype == MF_DTYPE_F32, p.bias_sums = bias_sums;
  p.weight_tiles = w.wanted, p.first = w.first, p.first2 = w.tiles1, p.pieces = w.pieces, p.per = w.per;
  p.one.m = 2 * F, p.one.n = C, p.input.m = (int)a->rows, p.input.n = C;
  if (a->grad_w_in) MF_MAP(weight_problem<T>(p.one, a, grad_pre, 2 * F, a->x, C, a->grad_w_in));
  if (a->grad_w_out) MF_MAP(weight_problem<T>(p.two, a, a->grad_y, O, a->act, F, a->grad_w_out));
  if (a->grad_x) {
    MF_MAP(map16<T>(&p.input.a, grad_pre, a->rows, 2 * F, 2 * F, 64));
    MF_MAP(map16<T>(&p.input.b, a->w_in, 2 * F, C, C, 64));
    MF_MAP(map16<T>(&p.input.out, a->grad_x, a->rows, C, C, 32));
  }
  const bool parts = w.pieces > 1;
  if (parts) {
    const long long dims[2] = {kTile, (long long)w.wanted * w.pieces * kTile}, strides[1] = {4 * kTile};
    MF_MAP(make_tensor_map(&p.pre, planes, MF_DTYPE_F32, 2, dims, strides, 32, 32));
  }
  const int input = a->grad_x ? tiles_of(a->rows, C, kTile) : 0;
  const Rounds r = rounds_of(w.wanted * w.pieces, w.per, input, input_blocks(a));
  const int others = input - r.tiles_ahead, rest = others % r.pairs;
  p.ahead = r.ahead, p.tiles_ahead = r.tiles_ahead;
  p.cut = rest == 0 || 2 * rest > r.pairs ? 1 : 4 * rest > r.pairs ? 2 : 4;
  p.whole = p.cut == 1 ? others : others - rest;
  p.tiles = p.whole + (others - p.whole) * p.cut;
  const int rc = launch_kernel<T, true, true, kGradients, 0>(p, r.pairs, stream, "gated_mlp gradients");
  if (rc != MF_OK || !parts) return rc;
  auto add = [&](auto* out1) {
    using TOut = std::remove_pointer_t<decltype(out1)>;
    launch_dependent(add_planes_kernel<T, TOut>, dim3(w.wanted, kTile / 4), dim3(256), 0, stream, planes, w, static_cast<TOut*>(a->grad_w_in), 2 * F, C,
                     static_cast<TOut*>(a->grad_w_out), O, F);
  };
  if (p.wide_out) add(static_cast<float*>(nullptr));
  else add(static_cast<T*>(nullptr));
  MF_CHECK_LAUNCH("add_planes_kernel");
  return MF_OK;
}

template <typename T>
int backward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const long long M = a->rows, C = a->dim, F = a->hidden, O = a->dim_out;
  size_t at[4];
  pieces(a, at);
  char* ws = static_cast<char*>(a->workspace);
  T* grad_pre = reinterpret_cast<T*>(ws + at[0]);
  float *planes = reinterpret_cast<float*>(ws + at[1]), *sums = reinterpret_cast<float*>(ws + at[2]);
  const bool biased = a->grad_b_in || a->grad_b_out;
  const BiasSums b = {a->grad_y, sums, biased ? reinterpret_cast<float*>(ws + at[3]) : nullptr, M, a->grad_b_out ? (int)O : 0, a->grad_b_in ? (int)(2 * F) : 0};
  int rc;
  if (forms_pre_gradient(a)) {
    Params p = common(M, F, O, waits);
    p.column_sums = a->grad_b_in ? sums : nullptr;
    p.exponents = exponents_of(a);
    MF_MAP(map16<T>(&p.one.a, a->grad_y, M, O, O, 64));
    MF_MAP(map16<T>(&p.one.b, a->w_out, O, F, F, 64));
    MF_MAP(map16<T>(&p.pre, a->pre, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.pre2, static_cast<const T*>(a->pre) + F, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.one.out, grad_pre, M, F, 2 * F, 32));
    MF_MAP(map16<T>(&p.out2, grad_pre + F, M, F, 2 * F, 32));
    cut_tiles<kGateGrad>(p);
    if ((rc = launch<T, false, true, kGateGrad>(p, a->activation, stream, "gated_mlp gate gradient")) != MF_OK) return rc;
  }
  if (a->grad_w_in || a->grad_w_out) {
    if ((rc = gradients<T>(a, grad_pre, planes, b, waits, stream)) != MF_OK) return rc;
  } else if (a->grad_x) {
    Params p = common(M, C, 2 * F, waits);
    MF_MAP(map16<T>(&p.one.a, grad_pre, M, 2 * F, 2 * F, 64));
    MF_MAP(map16<T>(&p.one.b, a->w_in, 2 * F, C, C, 64));
    if ((rc = store_product<T, true>(p, nullptr, static_cast<T*>(a->grad_x), nullptr, stream, "gated_mlp input gradient")) != MF_OK) return rc;
  }
  if (!biased) return MF_OK;
  if (!a->grad_w_in && !a->grad_w_out) {
    launch_dependent(bias_bands_kernel<T>, dim3(kBands / 2), dim3(64), 0, stream, b);
    MF_CHECK_LAUNCH("bias_bands_kernel");
  }
  const dim3 grid((b.n_in + b.n_out + 31) / 32);
  if (a->grad_dtype == MF_DTYPE_F32)
    launch_dependent(add_bias_bands_kernel<float>, grid, dim3(256), 0, stream, b, static_cast<float*>(a->grad_b_in), static_cast<float*>(a->grad_b_out));
  else launch_dependent(add_bias_bands_kernel<T>, grid, dim3(256), 0, stream, b, static_cast<T*>(a->grad_b_in), static_cast<T*>(a->grad_b_out));
  MF_CHECK_LAUNCH("add_bias_bands_kernel");
  return MF_OK;
}

int run_forward(const MfGatedMlpArgs* a, const BoundedWaits& waits, cudaStream_t stream) {
  const int rc = check(a);
  if (rc != MF_OK || a->rows == 0) return rc;
  MF_CHECK_ARG(a->y, "%s: null tensor", kName);
  if (gated_mlp_small(a) && waits.withheld < 0) return gated_mlp_small_forward(a, stream);
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
  const size_t need = pieces(a, at);
  if (need && (!a->workspace || a->workspace_bytes < need)) {
    set_error("%s: workspace too small (%zu bytes needed)", kName, need);
    return MF_ERR_WORKSPACE_TOO_SMALL;
  }
  return a->dtype == MF_DTYPE_BF16 ? backward<__nv_bfloat16>(a, waits, stream) : backward<__half>(a, waits, stream);
}

// Reads a status word and clears it in one step, so that an expired wait is reported once and none is lost.
__device__ int32_t g_taken_status;
__global__ void take_status_kernel(int word) { g_taken_status = atomicExch(&g_gemm_status[word], 0); }
int take_status(int word, int32_t* host_status, cudaStream_t stream) {
  static std::mutex one_at_a_time;  // (the word it goes through)
  const std::lock_guard<std::mutex> lock(one_at_a_time);
  take_status_kernel<<<1, 1, 0, stream>>>(word);
  MF_CHECK_LAUNCH("gated_mlp status read-back");
  cudaError_t e = cudaMemcpyFromSymbolAsync(host_status, g_taken_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "gated_mlp status read-back");
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" size_t mf_gated_mlp_pre_bytes(int64_t rows, int32_t hidden) {
  return rows < 0 || hidden < 1 ? 0 : gated_mlp_pre_values(rows, hidden) + (size_t)rows * ((hidden + 63) / 64) * 8;
}
extern "C" size_t mf_gated_mlp_fwd_workspace_bytes(const MfGatedMlpArgs* a) {
  if (!a || a->hidden < 1 || a->dim < 1 || a->dim_out < 1 || gated_mlp_small(a)) return 0;
  return slice_bytes(a->rows, a->dim_out, a->hidden);
}
extern "C" size_t mf_gated_mlp_bwd_workspace_bytes(const MfGatedMlpArgs* a) {
  if (!a || a->rows < 0 || a->hidden < 1 || a->dim < 1 || a->dim_out < 1) return 0;
  size_t at[4];
  return pieces(a, at);
}
extern "C" int mf_gated_mlp_fwd(const MfGatedMlpArgs* a, void* stream) { return run_forward(a, BoundedWaits{}, static_cast<cudaStream_t>(stream)); }
extern "C" int mf_gated_mlp_bwd(const MfGatedMlpArgs* a, void* stream) { return run_backward(a, BoundedWaits{}, static_cast<cudaStream_t>(stream)); }
extern "C" int mf_gated_mlp_status(int32_t* host_status, void* stream) {
  MF_CHECK_ARG(host_status != nullptr, "mf_gated_mlp_status: null pointer");
  return take_status(0, host_status, static_cast<cudaStream_t>(stream));
}
extern "C" int mf_selftest_gated_mlp_give_up(const MfGatedMlpArgs* a, int32_t backward, int32_t kind, int64_t limit_cycles, int32_t* host_status,
                                             void* stream) {
  MF_CHECK_ARG(a && kind >= 0 && kind <= 3, "mf_selftest_gated_mlp_give_up: bad argument");
  MF_CHECK_ARG(limit_cycles > 0 && limit_cycles <= kWaitLimitCycles, "mf_selftest_gated_mlp_give_up: the limit must lie in (0, 2^31] clocks");
  BoundedWaits waits;
  waits.limit = limit_cycles, waits.withheld = kind, waits.word = host_status != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = backward ? run_backward(a, waits, s) : run_forward(a, waits, s);
  return rc != MF_OK || !host_status ? rc : take_status(1, host_status, s);
}
