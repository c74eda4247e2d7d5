// Rotary positions: the channel pairs of every head turn by angle = position * frequency.
//
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos),   pair p of P = axes * pairs uses axis p / pairs and its own frequency;
//   half layout: a = x[p], b = x[p + P];   interleaved: a = x[2 p], b = x[2 p + 1];   channels from 2 P on are copied.
//
// The backward pass is the same rotation by the opposite angle.  Every value is read and written once: memory bounds it.  A block takes some
// tokens of one tensor, computes their cosines and sines once into shared memory, for all heads, and walks the rows (token, head) in
// the order in which they lie in memory, 16 bytes at a time where sizes, strides and addresses allow it, else 8, 4 or a single element.
//
// Angles are formed in turns in 64 bits, position * (frequency / 2 pi), and lose their whole turns there: a position of a million
// and a frequency of 1 would leave 4 digits of an angle in 32 bits.  What remains is at most half a turn: its sine and cosine are taken in
// 32 bits.
#include "common.cuh"

namespace mf {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kThreads = 256;

struct RotaryTensor {
  const void* in;
  void* out;
  int heads, rotates;
  long long in_batch, in_token, in_head, out_batch, out_token, out_head;
};
struct RotaryParams {
  double turns[kMaxPairs];  // frequency / 2 pi
  RotaryTensor tensor[3];
  const void* positions;
  long long position_batch;
  long long places;  // batch * tokens
  int tokens, head_dim, axes, pairs, position_type;
  int block_tokens;
  float amplitude, sign;
};

__device__ __forceinline__ double position_at(const RotaryParams& p, long long i) {
  switch (p.position_type) {
    case MF_POSITION_I32: return (double)static_cast<const int32_t*>(p.positions)[i];
    case MF_POSITION_I64: return (double)static_cast<const int64_t*>(p.positions)[i];
    case MF_POSITION_F32: return (double)static_cast<const float*>(p.positions)[i];
    default: return static_cast<const double*>(p.positions)[i];
  }
}

template <int kBytes>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

template <typename T, int kVec>
union Pack {
  typename Raw<sizeof(T) * kVec>::type raw;
  T v[kVec];
  __device__ Pack() {}
};
template <typename T, int kVec>
__device__ __forceinline__ Pack<T, kVec> load(const T* p) {
  Pack<T, kVec> r;
  r.raw = __ldg(reinterpret_cast<const typename Raw<sizeof(T) * kVec>::type*>(p));
  return r;
}
template <typename T, int kVec>
__device__ __forceinline__ void store(T* p, const Pack<T, kVec>& v) {
  *reinterpret_cast<typename Raw<sizeof(T) * kVec>::type*>(p) = v.raw;
}

// A unit is what a thread does of a row: kVec pairs of the half layout (two vectors), kVec / 2 pairs of the interleaved one (one vector;
// kVec 1: one pair, two elements), or a vector of the copied channels.
template <typename T, int kVec, bool kHalf>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 table[];  // (block_tokens, P): cosine, sine
  const RotaryTensor& x = p.tensor[blockIdx.y];
  const int P = p.axes * p.pairs;
  constexpr int kPairs = kHalf || kVec == 1 ? kVec : kVec / 2;  // of a rotating unit
  const long long first = (long long)blockIdx.x * p.block_tokens;
  const int count = (int)(p.places - first < p.block_tokens ? p.places - first : p.block_tokens);
  wait_for_previous();
  launch_dependents();
  if (x.rotates) {
    for (int i = threadIdx.x; i < count * P; i += kThreads) {
      const int token = i / P, pair = i - token * P;
      const long long place = first + token, b = place / p.tokens, n = place - b * p.tokens;
      double t = position_at(p, b * p.position_batch + n * p.axes + pair / p.pairs) * p.turns[pair];
      t -= rint(t);
      float s, c;
      sincospif(2.f * (float)t, &s, &c);
      table[i] = make_float2(p.amplitude * c, p.sign * p.amplitude * s);
    }
    __syncthreads();
  }
  const int rotating = P / kPairs, copied = (p.head_dim - 2 * P) / kVec, units = rotating + copied;
  const int rows = count * x.heads;
  const bool token_first = x.in_token < x.in_head;  // the rows of one head follow each other
  const int at_once = kThreads / units > 0 ? kThreads / units : 1;
  for (int u = threadIdx.x % units; u < units; u += kThreads) {  // (more units than threads: each takes several)
    const int j = units > kThreads ? 0 : threadIdx.x / units;
    if (j >= at_once) break;
#pragma unroll 2
    for (int r = j; r < rows; r += at_once) {
      const int head = token_first ? r / count : r % x.heads, token = token_first ? r - head * count : r / x.heads;
      const long long place = first + token, b = place / p.tokens, n = place - b * p.tokens;
      const T* in = static_cast<const T*>(x.in) + b * x.in_batch + n * x.in_token + head * x.in_head;
      T* out = static_cast<T*>(x.out) + b * x.out_batch + n * x.out_token + head * x.out_head;
      if (u >= rotating) {
        const int at = 2 * P + (u - rotating) * kVec;
        store<T, kVec>(out + at, load<T, kVec>(in + at));
        continue;
      }
      const float2* cs = table + token * P + u * kPairs;
      if constexpr (kHalf || kVec == 1) {
        const int at = kHalf ? u * kVec : 2 * u, other = kHalf ? at + P : at + 1;
        Pack<T, kVec> a = load<T, kVec>(in + at), c = load<T, kVec>(in + other);
        if (x.rotates) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const float va = to_f32<T>(a.v[e]), vc = to_f32<T>(c.v[e]);
            const float2 w = cs[e];
            a.v[e] = from_f32<T>(va * w.x - vc * w.y);
            c.v[e] = from_f32<T>(va * w.y + vc * w.x);
          }
        }
        store<T, kVec>(out + at, a);
        store<T, kVec>(out + other, c);
      } else {
        Pack<T, kVec> a = load<T, kVec>(in + u * kVec);
        if (x.rotates) {
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const float va = to_f32<T>(a.v[e]), vc = to_f32<T>(a.v[e + 1]);
            const float2 w = cs[e / 2];
            a.v[e] = from_f32<T>(va * w.x - vc * w.y);
            a.v[e + 1] = from_f32<T>(va * w.y + vc * w.x);
          }
        }
        store<T, kVec>(out + u * kVec, a);
      }
    }
  }
}

template <typename T, int kVec>
int launch(const RotaryParams& p, int tensors, bool half, cudaStream_t stream) {
  const long long blocks = (p.places + p.block_tokens - 1) / p.block_tokens;
  const dim3 grid((unsigned)blocks, (unsigned)tensors);
  const size_t smem = (size_t)p.block_tokens * p.axes * p.pairs * sizeof(float2);
  const cudaError_t e = half ? launch_dependent(rotary_kernel<T, kVec, true>, grid, dim3(kThreads), smem, stream, p)
                             : launch_dependent(rotary_kernel<T, kVec, false>, grid, dim3(kThreads), smem, stream, p);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "rotary_kernel");
}

template <typename T>
int launch_widest(const RotaryParams& p, int tensors, bool half, int vec, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch<T, 8>(p, tensors, half, stream);
  if (vec >= 4) return launch<T, 4>(p, tensors, half, stream);
  return vec == 2 ? launch<T, 2>(p, tensors, half, stream) : launch<T, 1>(p, tensors, half, stream);
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" int mf_rotary(const MfRotaryArgs* a, void* stream) {
  const char* name = "mf_rotary";
  MF_CHECK_ARG(a != nullptr, "%s: null argument struct", name);
  MF_CHECK_ARG(a->dtype == MF_DTYPE_F32 || a->dtype == MF_DTYPE_BF16 || a->dtype == MF_DTYPE_F16,
               "%s: only supports float16/bfloat16/float32 inputs, got dtype code %d", name, (int)a->dtype);
  MF_CHECK_ARG(a->batch >= 0 && a->tokens >= 0 && a->head_dim > 0, "%s: negative size", name);
  MF_CHECK_ARG(a->axes >= 1 && a->pairs >= 1 && a->axes <= kMaxPairs && a->pairs <= kMaxPairs && a->axes * a->pairs <= kMaxPairs,
               "%s: axes * pairs must lie in [1, %d], got %d * %d", name, kMaxPairs, (int)a->axes, (int)a->pairs);
  const int P = a->axes * a->pairs;
  MF_CHECK_ARG(2 * P <= a->head_dim, "%s: %d pairs need a head_dim of at least %d, got %d", name, P, 2 * P, (int)a->head_dim);
  MF_CHECK_ARG(a->layout == MF_ROTARY_HALF || a->layout == MF_ROTARY_INTERLEAVED, "%s: unknown layout code %d", name, (int)a->layout);
  MF_CHECK_ARG(a->position_type >= MF_POSITION_I32 && a->position_type <= MF_POSITION_F64, "%s: unknown position type %d", name, (int)a->position_type);
  MF_CHECK_ARG(a->tensors >= 1 && a->tensors <= 3, "%s: between one and three tensors, got %d", name, (int)a->tensors);
  MF_CHECK_ARG(a->frequencies != nullptr, "%s: null frequencies", name);
  const long long places = (long long)a->batch * a->tokens;
  RotaryParams p;
  for (int i = 0; i < P; ++i) p.turns[i] = a->frequencies[i] / 6.283185307179586476925286766559;
  const int size = a->dtype == MF_DTYPE_F32 ? 4 : 2;
  int vec = 16 / size, most_heads = 0;
  const bool half = a->layout == MF_ROTARY_HALF;
  auto fits = [&](long long elements) {
    while (vec > 1 && elements % vec) vec /= 2;
  };
  fits(half ? P : 2 * P);
  fits(a->head_dim - 2 * P);
  fits(a->head_dim);
  int used = 0;
  for (int i = 0; i < a->tensors; ++i) {
    const MfRotaryTensor& t = a->tensor[i];
    MF_CHECK_ARG(t.heads >= 0, "%s: negative size", name);
    if (t.heads == 0 || places == 0) continue;
    MF_CHECK_ARG(t.in && t.out, "%s: null tensor", name);
    MF_CHECK_ARG(reinterpret_cast<uintptr_t>(t.in) % size == 0 && reinterpret_cast<uintptr_t>(t.out) % size == 0, "%s: unaligned tensor", name);
    for (long long s : {(long long)t.in_batch, (long long)t.in_token, (long long)t.in_head, (long long)t.out_batch, (long long)t.out_token, (long long)t.out_head,
                        (long long)(reinterpret_cast<uintptr_t>(t.in) / size), (long long)(reinterpret_cast<uintptr_t>(t.out) / size)})
      fits(s);
    p.tensor[used++] = {t.in, t.out, t.heads, t.rotates, t.in_batch, t.in_token, t.in_head, t.out_batch, t.out_token, t.out_head};
    if (t.heads > most_heads) most_heads = t.heads;
  }
  if (used == 0) return MF_OK;
  MF_CHECK_ARG(a->positions != nullptr, "%s: null positions", name);
  p.positions = a->positions, p.position_batch = a->position_batch, p.places = places;
  p.tokens = a->tokens, p.head_dim = a->head_dim, p.axes = a->axes, p.pairs = a->pairs, p.position_type = a->position_type;
  p.amplitude = a->amplitude, p.sign = a->inverse ? -1.f : 1.f;
  // up to 32 tokens a block, so that each head's stretch of a tensor is long, while there are four blocks for every SM
  p.block_tokens = 32;
  while (p.block_tokens > 1 && (places + p.block_tokens - 1) / p.block_tokens * used < 4 * 148) p.block_tokens /= 2;
  const long long blocks = (places + p.block_tokens - 1) / p.block_tokens;
  MF_CHECK_ARG(blocks < (1ll << 31), "%s: batch * tokens above 2^36", name);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case MF_DTYPE_F32: return launch_widest<float>(p, used, half, vec, s);
    case MF_DTYPE_BF16: return launch_widest<__nv_bfloat16>(p, used, half, vec, s);
    default: return launch_widest<__half>(p, used, half, vec, s);
  }
}
