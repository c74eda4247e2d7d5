// Rotary positions: the channel pairs of every head turn by angle = position * frequency.
//
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos),   pair p of P = axes * pairs uses axis p / pairs and its own frequency;
//   half layout: a = x[p], b = x[p + P];   interleaved: a = x[2 p], b = x[2 p + 1];   channels from 2 P on are copied.
//
// The backward pass is the same rotation by the opposite angle.  Every value is read and written once: memory bounds it.  A warp takes a few
// tokens: its lanes form the tokens' cosines and sines, once for all heads of all tensors, into a table of the warp in shared memory, and
// then move the tokens' rows, 16 bytes at a time where sizes, strides and addresses allow it, else 8, 4 or a single element.  Warps wait
// for nobody, so that one's arithmetic hides behind the others' loads.  Copies reach 6.5 TB/s; 20 heads of 128, 32 771 tokens, fp32: 117 us,
// 5.7 TB/s; 32 x 8 + 8 interleaved heads of 64, 4096 tokens, bf16: 99 us, 5.4; packed projections of 1024 x 29 tokens, three axes, bf16: 44 us,
// 4.1, where the angles of four tokens come before each warp's 12 KB.  (Its first loads before the angles: 50 us; that takes 117 registers.)
//
// Angles are formed in turns in 64 bits, position * (frequency / 2 pi), and lose their whole turns there: a position of a million
// and a frequency of 1 would leave 4 digits of an angle in 32 bits.  What remains is at most half a turn: its sine and cosine are taken in
// 32 bits.
#include "common.cuh"

namespace mf {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kWarps = 4;
constexpr int kBatch = 4;  // items of a lane in flight

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
  int batch, tokens, head_dim, axes, pairs, position_type;
  int warp_tokens, tensors;
  int parts;  // warps that share a token's heads (gridDim.y)
  float amplitude, sign;
  int half, piece;
  int narrow;  // offsets within a warp's tokens fit 32 bits
};

__device__ __forceinline__ double position_at(const RotaryParams& p, long long i) {
  switch (p.position_type) {
    case MF_POSITION_I32: return (double)static_cast<const int32_t*>(p.positions)[i];
    case MF_POSITION_I64: return (double)static_cast<const int64_t*>(p.positions)[i];
    case MF_POSITION_F32: return (double)static_cast<const float*>(p.positions)[i];
    default: return static_cast<const double*>(p.positions)[i];
  }
}

// kVec elements as 32-bit registers.  (Plain loads: the kernel before may still write what they read when this one begins, and a load that is
// marked as read-only may be moved above the wait for it.)
template <typename T, int kVec>
struct Vec {
  static constexpr int kBytes = sizeof(T) * kVec;
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 16) {
      uint4 v;  // (stays behind the wait as well, but lets the stores of earlier items pass: interleaved heads of 64 108 -> 101 us)
      asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
  __device__ __forceinline__ void get(float (&v)[kVec]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = __uint_as_float(w[e]);
    } else if constexpr (kVec == 1) {
      v[0] = unpack2<T>(w[0]).x;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const float2 f = unpack2<T>(w[e / 2]);
        v[e] = f.x, v[e + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[kVec]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = __float_as_uint(v[e]);
    } else if constexpr (kVec == 1) {
      w[0] = pack2<T>(v[0], 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e += 2) w[e / 2] = pack2<T>(v[e], v[e + 1]);
    }
  }
};

// cos and sin of kPairs pairs from one on, in 16-byte loads where there are four: P is a multiple of kPairs then
template <int kPairs>
__device__ __forceinline__ void angles(const float* cosine, const float* sine, float (&c)[kPairs], float (&s)[kPairs]) {
  if constexpr (kPairs >= 4) {
#pragma unroll
    for (int e = 0; e < kPairs; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(cosine + e), w = *reinterpret_cast<const float4*>(sine + e);
      c[e] = v.x, c[e + 1] = v.y, c[e + 2] = v.z, c[e + 3] = v.w;
      s[e] = w.x, s[e + 1] = w.y, s[e + 2] = w.z, s[e + 3] = w.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPairs; ++e) c[e] = cosine[e], s[e] = sine[e];
  }
}

// The partners of the channels from `at` on, `from` their address: P channels further on or back, in pieces of 1, 2 or 4 elements which lie
// within one half each.  Channels from 2 P on have none.
template <typename T, int kVec, int kPiece>
__device__ __forceinline__ void partners_of(Vec<T, kVec>& c, const T* from, int at, int P) {
  constexpr int kWords = sizeof(T) * kPiece / 4 ? sizeof(T) * kPiece / 4 : 1;
  uint32_t half = 0;
#pragma unroll
  for (int e = 0; e < kVec; e += kPiece) {
    Vec<T, kPiece> v;
#pragma unroll
    for (int w = 0; w < kWords; ++w) v.w[w] = 0;
    if (at + e < 2 * P) v.load(from + e + (at + e < P ? P : -P));
    if constexpr (sizeof(T) * kPiece == 2) {
      if (e % 2 == 0) half = v.w[0];
      else c.w[e / 2] = half | v.w[0] << 16;
    } else {
#pragma unroll
      for (int w = 0; w < kWords; ++w) c.w[e / kPiece * kWords + w] = v.w[w];
    }
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void partners(Vec<T, kVec>& c, const T* from, int at, int P, int piece) {
  if (kVec > 4 && piece == 4) partners_of<T, kVec, kVec < 4 ? kVec : 4>(c, from, at, P);
  else if (kVec > 2 && piece == 2) partners_of<T, kVec, 2>(c, from, at, P);
  else partners_of<T, kVec, 1>(c, from, at, P);
}

// What an item of a lane is:
//   kHalves       kVec pairs of the half layout, two vectors; or a vector of the copied channels (P a multiple of kVec)
//   kHalvesMixed  a vector, whose partners are fetched in pieces of `piece` elements, the power of two in P (they come from L1)
//   kNeighbours   a vector of kVec / 2 pairs of the interleaved layout
//   kSingle       a pair of either layout, element by element
enum Mode { kHalves, kHalvesMixed, kNeighbours, kSingle };

template <typename T, int kVec, Mode kMode>
__global__ void __launch_bounds__(32 * kWarps) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(16) float tables[];  // (warp, cosine | sine, warp_tokens, P)
  constexpr bool kTwo = kMode == kHalves || kMode == kSingle;  // a rotating item is two vectors
  constexpr int kPairs = kMode == kNeighbours ? kVec / 2 : kVec;
  constexpr int kInFlight = kMode == kHalvesMixed ? 2 : kBatch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = p.axes * p.pairs, rotating = kMode == kHalvesMixed ? 2 * P / kVec + 1 : (P + kPairs - 1) / kPairs;
  const int units = kTwo ? rotating + (p.head_dim - 2 * P) / kVec : p.head_dim / kVec;
  // tokens of one batch entry
  const int tiles = (p.tokens + p.warp_tokens - 1) / p.warp_tokens;
  const long long tile = (long long)blockIdx.x * kWarps + warp;
  const int b = tile <= 0x7fffffffll ? (int)tile / tiles : (int)(tile / tiles), n0 = (int)(tile - (long long)b * tiles) * p.warp_tokens;
  const int count = b < p.batch ? min(p.tokens - n0, p.warp_tokens) : 0;
  float* cosine = tables + warp * 2 * p.warp_tokens * P;
  float* sine = cosine + p.warp_tokens * P;
  launch_dependents();
  wait_for_previous();
  const long long at0 = b * p.position_batch + (long long)n0 * p.axes;
  for (int pair = lane; pair < P; pair += 32) {
    const double frequency = p.turns[pair];
    const int axis = p.axes == 1 ? 0 : pair / p.pairs;
    for (int t = 0; t < count; ++t) {
      double turns = position_at(p, at0 + t * p.axes + axis) * frequency;
      turns -= rint(turns);
      float s, c;
      if constexpr (sizeof(T) == 4) {
        sincospif(2.f * (float)turns, &s, &c);
      } else {  // 2^-21 of a pair's length, which is rounded to 2^-9 or 2^-12 of the value
        const float angle = 6.283185307179586f * (float)turns;
        s = __sinf(angle), c = __cosf(angle);
      }
      cosine[t * P + pair] = p.amplitude * c, sine[t * P + pair] = p.sign * p.amplitude * s;
    }
  }
  __syncwarp();
  for (int which = 0; which < p.tensors; ++which) {
    const RotaryTensor& x = p.tensor[which];
    const T* in = static_cast<const T*>(x.in) + b * x.in_batch + n0 * x.in_token;
    T* out = static_cast<T*>(x.out) + b * x.out_batch + n0 * x.out_token;
    // (token, head, unit) of this lane's items, 32 * parts further on each time
    const int h_units = x.heads * units, total = count * h_units, step = 32 * p.parts;
    int i = 32 * blockIdx.y + lane;
    int token = i / h_units, head = (i - token * h_units) / units, u = i - token * h_units - head * units;
    const int step_t = step / h_units, step_h = (step - step_t * h_units) / units, step_u = step - step_t * h_units - step_h * units;
    while (i < total) {
      Vec<T, kVec> a[kInFlight], c[kInFlight];
      T* to[kInFlight];
      int angle[kInFlight], other[kInFlight];  // the first angle, -1: copied; distance of the second vector, 0: one, -1: no item
      int channel[kInFlight];
#pragma unroll
      for (int k = 0; k < kInFlight; ++k) {
        other[k] = -1;
        if (i < total) {
          const bool turns = u < rotating;
          const int at = !kTwo || (kMode == kHalves && turns) ? u * kVec : turns ? (p.half ? u : 2 * u) : 2 * P + (u - rotating) * kVec;
          other[k] = kTwo && turns ? (kMode == kHalves || p.half ? P : 1) : 0;
          angle[k] = turns && x.rotates ? token * P + (kMode == kHalvesMixed ? 0 : u * kPairs) : -1;
          channel[k] = at;
          const T* from;
          if (p.narrow) {
            from = in + (token * (int)x.in_token + head * (int)x.in_head + at);
            to[k] = out + (token * (int)x.out_token + head * (int)x.out_head + at);
          } else {
            from = in + token * x.in_token + head * x.in_head + at;
            to[k] = out + token * x.out_token + head * x.out_head + at;
          }
          a[k].load(from);
          if (kTwo && other[k]) c[k].load(from + other[k]);
          if constexpr (kMode == kHalvesMixed)
            if (angle[k] >= 0) partners(c[k], from, at, P, p.piece);
        }
        i += step, token += step_t, head += step_h, u += step_u;
        if (u >= units) u -= units, ++head;
        if (head >= x.heads) head -= x.heads, ++token;
      }
#pragma unroll
      for (int k = 0; k < kInFlight; ++k) {
        if (other[k] < 0) break;
        if (angle[k] >= 0) {
          float cs[kPairs], sn[kPairs], va[kVec];
          a[k].get(va);
          if constexpr (kMode == kHalvesMixed) {
            float vc[kVec];
            c[k].get(vc);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              const int at = channel[k] + e;
              if (at < 2 * P) {
                const int pair = angle[k] + (at < P ? at : at - P);
                va[e] = at < P ? va[e] * cosine[pair] - vc[e] * sine[pair] : vc[e] * sine[pair] + va[e] * cosine[pair];
              }
            }
          } else if constexpr (kTwo) {
            float vc[kVec];
            c[k].get(vc);
            angles<kPairs>(cosine + angle[k], sine + angle[k], cs, sn);
            if constexpr (kVec >= 2) {
#pragma unroll
              for (int e = 0; e < kVec; e += 2) {
                const float2 v = make_float2(va[e], va[e + 1]), w = make_float2(vc[e], vc[e + 1]);
                const float2 co = make_float2(cs[e], cs[e + 1]), si = make_float2(sn[e], sn[e + 1]);
                const float2 y = fma2(v, si, mul2(w, co)), z = mul2(w, si);
                const float2 r = fma2(v, co, make_float2(-z.x, -z.y));
                va[e] = r.x, va[e + 1] = r.y, vc[e] = y.x, vc[e + 1] = y.y;
              }
            } else {
              const float v = va[0], w = vc[0];
              va[0] = v * cs[0] - w * sn[0], vc[0] = v * sn[0] + w * cs[0];
            }
            c[k].set(vc);
          } else {
            if (P % kPairs == 0) {  // a vector turns whole
              angles<kPairs>(cosine + angle[k], sine + angle[k], cs, sn);
#pragma unroll
              for (int e = 0; e < kVec; e += 2) {
                const float v = va[e], w = va[e + 1];
                va[e] = v * cs[e / 2] - w * sn[e / 2], va[e + 1] = v * sn[e / 2] + w * cs[e / 2];
              }
            } else {  // (the table has room for a vector behind its last pair)
#pragma unroll
              for (int e = 0; e < kVec; e += 2) {
                const float v = va[e], w = va[e + 1], co = cosine[angle[k] + e / 2], si = sine[angle[k] + e / 2];
                if (channel[k] / 2 + e / 2 < P) va[e] = v * co - w * si, va[e + 1] = v * si + w * co;
              }
            }
          }
          a[k].set(va);
        }
        a[k].store(to[k]);
        if (kTwo && other[k]) c[k].store(to[k] + other[k]);
      }
    }
  }
}

template <typename T, int kVec, Mode kMode>
int launch(RotaryParams& p, cudaStream_t stream) {
  const int P = p.axes * p.pairs;
  const int units = kMode == kHalves || kMode == kSingle ? P / kVec + (p.head_dim - 2 * P) / kVec : p.head_dim / kVec;
  // Up to eight tokens a warp while that leaves 32 warps for every SM (measured with 16, 32 and 64: 1024 x 29 tokens of 16 rotated and 8
  // copied heads of 64, three axes, bf16, 49.3, 47.8 and 54.2 us; 32 771 tokens of 20 heads of 128, fp32, 133, 119 and 117 us); with few
  // tokens, a token's heads go to several warps.
  p.warp_tokens = 8;
  auto warps = [&] { return (long long)p.batch * ((p.tokens + p.warp_tokens - 1) / p.warp_tokens); };
  while (p.warp_tokens > 1 && (warps() < 32 * 148 || p.warp_tokens >= 2 * p.tokens)) p.warp_tokens /= 2;
  const long long blocks = (warps() + kWarps - 1) / kWarps;
  int heads = 0;
  for (int i = 0; i < p.tensors; ++i) heads = heads > p.tensor[i].heads ? heads : p.tensor[i].heads;
  p.narrow = 1;
  for (int i = 0; i < p.tensors; ++i) {
    const RotaryTensor& t = p.tensor[i];
    const long long strides[2][2] = {{t.in_token, t.in_head}, {t.out_token, t.out_head}};
    for (const auto& s : strides) {
      const double reach = (double)p.warp_tokens * (double)(s[0] < 0 ? -s[0] : s[0]) + (double)t.heads * (double)(s[1] < 0 ? -s[1] : s[1]) + p.head_dim;
      if (reach > 2147483647.) p.narrow = 0;
    }
  }
  const long long most = ((long long)p.warp_tokens * heads * units + 31) / 32;
  long long parts = 16 * 148 / (blocks * kWarps);
  p.parts = (int)(parts < 1 ? 1 : parts > most ? most : parts > 64 ? 64 : parts);
  MF_CHECK_ARG(blocks < (1ll << 31), "mf_rotary: batch * tokens above 2^33");
  const dim3 grid((unsigned)blocks, (unsigned)p.parts);
  const size_t smem = (size_t)(kWarps * 2 * p.warp_tokens * P + kVec) * sizeof(float);
  const cudaError_t e = launch_dependent(rotary_kernel<T, kVec, kMode>, grid, dim3(32 * kWarps), smem, stream, p);
  return e == cudaSuccess ? MF_OK : cuda_error(e, "rotary_kernel");
}

// `vec` elements at a time: what head_dim, strides and addresses are multiples of
template <typename T, int kVec>
int launch_mode(RotaryParams& p, int vec, cudaStream_t stream) {
  if constexpr (kVec > 1) {
    if (vec < kVec) return launch_mode<T, kVec / 2>(p, vec, stream);
    if (!p.half) return launch<T, kVec, kNeighbours>(p, stream);
    const int P = p.axes * p.pairs;
    if (P % kVec == 0) return launch<T, kVec, kHalves>(p, stream);
    p.piece = P % 4 == 0 ? 4 : P % 2 == 0 ? 2 : 1;
    return launch<T, kVec, kHalvesMixed>(p, stream);
  } else {
    return launch<T, 1, kSingle>(p, stream);
  }
}

// Whether b's heads lie behind a's, as queries and keys of a packed projection do: one tensor then, whose last round of a warp's lanes is
// fuller (1024 x 29 tokens, three axes: 46 -> 44 us).
bool continues(const RotaryTensor& a, const RotaryTensor& b, int size) {
  return (a.rotates != 0) == (b.rotates != 0) && a.in_batch == b.in_batch && a.in_token == b.in_token && a.in_head == b.in_head && a.out_batch == b.out_batch &&
         a.out_token == b.out_token && a.out_head == b.out_head && static_cast<const char*>(a.in) + a.heads * a.in_head * size == b.in &&
         static_cast<char*>(a.out) + a.heads * a.out_head * size == b.out;
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
  int vec = 16 / size;
  auto fits = [&](long long elements) {
    while (vec > 1 && elements % vec) vec /= 2;
  };
  fits(a->head_dim);
  int used = 0;
  for (int i = 0; i < a->tensors; ++i) {
    const MfRotaryTensor& t = a->tensor[i];
    MF_CHECK_ARG(t.heads >= 0, "%s: negative size", name);
    // (a warp counts the pieces of its eight tokens' heads in 32 bits)
    MF_CHECK_ARG((long long)t.heads * a->head_dim <= 1 << 27, "%s: %d heads of %d channels, more than 2^27 elements a token", name, (int)t.heads,
                 (int)a->head_dim);
    if (t.heads == 0 || places == 0) continue;
    MF_CHECK_ARG(t.in && t.out, "%s: null tensor", name);
    MF_CHECK_ARG(reinterpret_cast<uintptr_t>(t.in) % size == 0 && reinterpret_cast<uintptr_t>(t.out) % size == 0, "%s: unaligned tensor", name);
    for (long long s : {(long long)t.in_batch, (long long)t.in_token, (long long)t.in_head, (long long)t.out_batch, (long long)t.out_token, (long long)t.out_head,
                        (long long)(reinterpret_cast<uintptr_t>(t.in) / size), (long long)(reinterpret_cast<uintptr_t>(t.out) / size)})
      fits(s);
    const RotaryTensor next = {t.in, t.out, t.heads, t.rotates, t.in_batch, t.in_token, t.in_head, t.out_batch, t.out_token, t.out_head};
    if (used && continues(p.tensor[used - 1], next, size) && (long long)(p.tensor[used - 1].heads + t.heads) * a->head_dim <= 1 << 27) p.tensor[used - 1].heads += t.heads;
    else p.tensor[used++] = next;
  }
  if (used == 0) return MF_OK;
  MF_CHECK_ARG(a->positions != nullptr, "%s: null positions", name);
  p.positions = a->positions, p.position_batch = a->position_batch;
  p.batch = a->batch, p.tokens = a->tokens, p.head_dim = a->head_dim, p.axes = a->axes, p.pairs = a->pairs, p.position_type = a->position_type;
  p.half = a->layout == MF_ROTARY_HALF, p.piece = 1;
  p.tensors = used, p.amplitude = a->amplitude, p.sign = a->inverse ? -1.f : 1.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case MF_DTYPE_F32: return launch_mode<float, 4>(p, vec, s);
    case MF_DTYPE_BF16: return launch_mode<__nv_bfloat16, 8>(p, vec, s);
    default: return launch_mode<__half, 8>(p, vec, s);
  }
}
