// Rotary positions of queries and keys (gfx950).
//
// Pair i of a head's first `rotary` columns is turned by the angle position *
// freq[i]:  (a, b) -> A (a cos - b sin, a sin + b cos); the gradient is the turn
// by the negative angle with the same A.  Pairs are columns (2 i, 2 i + 1)
// (interleaved) or (i, i + rotary / 2); columns past `rotary` are copied.
//
// Memory bound: every value is read and written once, 16 bytes a lane.  The
// angles of a token are the same for all its heads, so a workgroup forms them
// once, in LDS, for the tokens it turns, one thread a pair.  An angle is position
// * freq / 2 pi in fp64 (at position 2^20 right to 2^-33 turns), of which the whole
// turns are dropped before the rest, half a turn at most, is rounded to fp32: 2^-26
// turns, where an fp32 product would be off by 2^-7.  Products are fp32, rounded once.
#include "mfma_tiles.h"

using namespace tcfp;

namespace {

constexpr int kThreads = 256;

struct Rotary {
  const void* x[2];
  void* y[2];
  int64_t token[2], head[2];  // strides of x in elements
  int heads[2];
  const int64_t* positions;
  const double* freqs;
  int64_t tokens;
  int dim, pairs;
  int per_block;  // tokens
  float amplitude, sign;
};

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static TCFP_DEV void load(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static TCFP_DEV void store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
  static TCFP_DEV float get(float v) { return v; }
  static TCFP_DEV float put(float v) { return v; }
};
template <>
struct Vec<uint16_t> {
  static constexpr int N = 8;
  static TCFP_DEV void load(const uint16_t* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
  static TCFP_DEV void store(uint16_t* p, const float* v) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]),
                                              pack2(v[4], v[5]), pack2(v[6], v[7]));
  }
  static TCFP_DEV float get(uint16_t v) { return bf16_to_f32(v); }
  static TCFP_DEV uint16_t put(float v) { return f32_to_bf16_rne(v); }
};

// VEC: the pairs of a head are whole 16-byte vectors (interleaved), or either
// half of them is; otherwise a thread turns one pair and copies one column at a
// time.
template <typename T, bool INTER, bool VEC>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Rotary r) {
  extern __shared__ float2 turn[];  // [token of the block][pair]: cos, sin
  using V = Vec<T>;
  const int64_t t0 = int64_t(blockIdx.x) * r.per_block;
  const int here = int(min(int64_t(r.per_block), r.tokens - t0));
  for (int i = threadIdx.x; i < here * r.pairs; i += kThreads) {
    const int t = i / r.pairs, p = i - t * r.pairs;
    double turns = double(r.positions[t0 + t]) * (r.freqs[p] * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * float(turns), &s, &c);
    turn[i] = make_float2(c * r.amplitude, s * r.amplitude * r.sign);
  }
  __syncthreads();
  const int heads = r.heads[0] + r.heads[1], rotary = 2 * r.pairs;
  // a head's work items: turned ones first, then copies
  constexpr int N = VEC ? V::N : 1;
  const int turned = !VEC ? r.pairs : INTER ? rotary / N : r.pairs / N;
  const int items = turned + (r.dim - rotary) / N;
  for (int i = threadIdx.x; i < here * heads * items; i += kThreads) {
    const int e = i % items, th = i / items, t = th / heads, hh = th - t * heads;
    const int which = hh >= r.heads[0], h = which ? hh - r.heads[0] : hh;
    const T* x = static_cast<const T*>(r.x[which]) + (t0 + t) * r.token[which] + h * r.head[which];
    T* y = static_cast<T*>(r.y[which]) + ((t0 + t) * r.heads[which] + h) * r.dim;
    const float2* cs = turn + t * r.pairs;
    if (e >= turned) {
      const int at = rotary + (e - turned) * N;
      if constexpr (VEC)
        *reinterpret_cast<uint4*>(y + at) = *reinterpret_cast<const uint4*>(x + at);
      else y[at] = x[at];
      continue;
    }
    if constexpr (VEC && INTER) {
      float v[N];
      V::load(x + e * N, v);
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const float2 c = cs[e * (N / 2) + j];
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = a * c.x - b * c.y;
        v[2 * j + 1] = a * c.y + b * c.x;
      }
      V::store(y + e * N, v);
    } else if constexpr (VEC) {
      float a[N], b[N];
      V::load(x + e * N, a);
      V::load(x + r.pairs + e * N, b);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 c = cs[e * N + j];
        const float p = a[j], q = b[j];
        a[j] = p * c.x - q * c.y;
        b[j] = p * c.y + q * c.x;
      }
      V::store(y + e * N, a);
      V::store(y + r.pairs + e * N, b);
    } else {
      const int at = INTER ? 2 * e : e, to = INTER ? at + 1 : at + r.pairs;
      const float a = V::get(x[at]), b = V::get(x[to]);
      const float2 c = cs[e];
      y[at] = V::put(a * c.x - b * c.y);
      y[to] = V::put(a * c.y + b * c.x);
    }
  }
}

constexpr int kMostPairs = 2048;  // LDS: 16 KiB of angles a token

}  // namespace

extern "C" int tcfp_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                           int q_heads, const void* k, int64_t k_token_stride,
                           int64_t k_head_stride, int k_heads, int dtype, int64_t tokens, int dim,
                           const int64_t* positions, const double* freqs, int rotary,
                           int interleaved, float amplitude, int inverse, void* q_out, void* k_out,
                           void* stream) {
  if (tokens < 0 || q_heads < 0 || k_heads < 0 || q_heads > 65535 || k_heads > 65535 || dim < 2 ||
      dim > 65536 || rotary < 2 || rotary % 2 || rotary > dim || rotary / 2 > kMostPairs)
    return TCFP_ERR_SHAPE;
  if (dtype != TCFP_DTYPE_F32 && dtype != TCFP_DTYPE_BF16) return TCFP_ERR_DTYPE;
  if (tokens == 0 || q_heads + k_heads == 0) return TCFP_OK;
  Rotary r{};
  r.x[0] = q; r.x[1] = k;
  r.y[0] = q_out; r.y[1] = k_out;
  r.token[0] = q_token_stride; r.token[1] = k_token_stride;
  r.head[0] = q_head_stride; r.head[1] = k_head_stride;
  r.heads[0] = q_heads; r.heads[1] = k_heads;
  r.positions = positions;
  r.freqs = freqs;
  r.tokens = tokens;
  r.dim = dim;
  r.pairs = rotary / 2;
  r.amplitude = amplitude;
  r.sign = inverse ? -1.0f : 1.0f;
  // whole 16-byte vectors everywhere, or one pair at a time
  const int n = dtype == TCFP_DTYPE_F32 ? 4 : 8;
  bool vec = (interleaved ? rotary : r.pairs) % n == 0 && (dim - rotary) % n == 0;
  for (int i = 0; i < 2; ++i)
    if (r.heads[i])
      vec = vec && (reinterpret_cast<uintptr_t>(r.x[i]) & 15) == 0 &&
            (reinterpret_cast<uintptr_t>(r.y[i]) & 15) == 0 && r.token[i] % n == 0 &&
            r.head[i] % n == 0;
  // A workgroup takes one token where there are few, so that they spread over the
  // card, else four, whose angles keep its threads busy.
  r.per_block = tokens < 1024 || r.pairs > kMostPairs / 4 ? 1 : 4;
  const int64_t blocks = (tokens + r.per_block - 1) / r.per_block;
  if (!grid_x_fits(blocks, kThreads) ||
      int64_t(r.per_block) * (q_heads + k_heads) * dim > INT32_MAX)
    return TCFP_ERR_SHAPE;
  const auto st = static_cast<hipStream_t>(stream);
  const size_t lds = size_t(r.per_block) * r.pairs * sizeof(float2);
#define TCFP_ROTARY(T, I, V) \
  rotary_kernel<T, I, V><<<unsigned(blocks), kThreads, lds, st>>>(r)
#define TCFP_ROTARY_T(T)                                            \
  do {                                                              \
    if (interleaved) {                                              \
      if (vec) TCFP_ROTARY(T, true, true); else TCFP_ROTARY(T, true, false);   \
    } else {                                                        \
      if (vec) TCFP_ROTARY(T, false, true); else TCFP_ROTARY(T, false, false); \
    }                                                               \
  } while (0)
  if (dtype == TCFP_DTYPE_F32) TCFP_ROTARY_T(float); else TCFP_ROTARY_T(uint16_t);
#undef TCFP_ROTARY_T
#undef TCFP_ROTARY
  return hipGetLastError() == hipSuccess ? TCFP_OK : TCFP_ERR_HIP;
}
