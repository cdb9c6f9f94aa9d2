// Paged K/V cache in E4M3 codes with one power-of-two exponent per token and
// head, and attention of new tokens over it, for gfx950.
//
//   codes [num_pages, kv_heads, page_size, dim], exps [num_pages, kv_heads,
//   page_size]: the keys of one page and head are one contiguous run, so a
//   tile of keys is read in whole lines whatever the number of heads.
#include <algorithm>

#include "common.h"

using namespace tcfp;

namespace {

constexpr int kThreads = 256;

inline int launch_status() { return hipGetLastError() == hipSuccess ? TCFP_OK : TCFP_ERR_HIP; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int log2i(int v) { return 31 - __builtin_clz(unsigned(v)); }

bool cache_ok(int64_t num_pages, int page_size, int kv_heads, int dim) {
  return num_pages >= 0 && num_pages <= INT32_MAX && kv_heads > 0 && kv_heads <= 65535 &&
         (dim == 64 || dim == 128 || dim == 256) && page_size >= 16 && page_size <= 1024 &&
         (page_size & (page_size - 1)) == 0;
}

TCFP_DEV void load8(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
TCFP_DEV void load8(const uint16_t* p, float* v) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
TCFP_DEV void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
TCFP_DEV uint32_t pack_bf16(float a, float b) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, r);
}
TCFP_DEV void store8(uint16_t* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                            pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// ---- the cache ---------------------------------------------------------------

struct Pool {
  uint8_t* codes[2];  // K, V
  int8_t* exps[2];
  int64_t slots;      // num_pages * page_size
  int heads;
  int page_bits;
};

// Place of a slot and head in exps (and, times dim, in codes).
TCFP_DEV int64_t place_of(const Pool& p, int64_t slot, int head) {
  const int64_t page = slot >> p.page_bits;
  const int off = int(slot) & ((1 << p.page_bits) - 1);
  return ((page * p.heads + head) << p.page_bits) + off;
}

struct Strided {
  const void* p[2];
  int64_t token[2], head[2];
};

// DIM / 8 lanes a (token, head), 8 values each; blockIdx.y: K or V.
template <typename T, int DIM>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(Strided x, Pool pool,
                                                               const int64_t* slots,
                                                               int64_t items) {
  constexpr int L = DIM / 8;
  const int64_t item = int64_t(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  if (item >= items) return;
  const int64_t t = item / pool.heads;
  const int head = int(item - t * pool.heads), li = threadIdx.x % L, kv = blockIdx.y;
  const int64_t slot = slots[t];
  const bool live = slot >= 0 && slot < pool.slots;
  float v[8];
  load8(static_cast<const T*>(x.p[kv]) + t * x.token[kv] + head * x.head[kv] + li * 8, v);
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = absbits(v[j]);
    if (b >= 0x7F800000u) v[j] = __uint_as_float(0x7FC00000u);  // no finite value: NaN
    else a = umax(a, b);
  }
  a = seg_umax<L>(a);
  const int e = block_exponent(__uint_as_float(a), kE4M3Max);
  const float mul = exp2i(-e);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = clampf(v[j] * mul, kE4M3Max);
  if (!live) return;
  const int64_t at = place_of(pool, slot, head);
  const uint2 w = make_uint2(cvt4_fp8<TCFP_FP8_E4M3>(v[0], v[1], v[2], v[3]),
                             cvt4_fp8<TCFP_FP8_E4M3>(v[4], v[5], v[6], v[7]));
  *reinterpret_cast<uint2*>(pool.codes[kv] + at * DIM + li * 8) = w;
  if (li == 0) pool.exps[kv][at] = int8_t(e);
}

template <typename T, int DIM>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(Pool pool, const int64_t* slots,
                                                              int64_t items, T* k, T* v_out) {
  constexpr int L = DIM / 8;
  const int64_t item = int64_t(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  if (item >= items) return;
  const int64_t t = item / pool.heads;
  const int head = int(item - t * pool.heads), li = threadIdx.x % L, kv = blockIdx.y;
  const int64_t slot = slots[t];
  float v[8] = {};
  if (slot >= 0 && slot < pool.slots) {
    const int64_t at = place_of(pool, slot, head);
    const uint2 w = *reinterpret_cast<const uint2*>(pool.codes[kv] + at * DIM + li * 8);
    const int e = pool.exps[kv][at];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = ldexpf(e4m3_to_f32(w.x >> (8 * j)), e);
      v[4 + j] = ldexpf(e4m3_to_f32(w.y >> (8 * j)), e);
    }
  }
  store8((kv ? v_out : k) + item * DIM + li * 8, v);
}

// ---- attention ---------------------------------------------------------------

struct Attend {
  const uint16_t* q;
  int64_t q_token, q_head;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const int8_t* k_exps;
  const int8_t* v_exps;
  int64_t num_pages;
  int page_bits;
  int kv_heads;
  const int32_t* table;
  int64_t table_stride;
  int64_t table_keys;  // keys that a row of the table spans
  const int32_t* seq_lens;
  const int32_t* starts;
  int64_t batch;
  int64_t tokens;
  int heads;
  int group;  // heads / kv_heads
  float scale;
  int causal;
  int64_t window;
  uint16_t* out;
};

// One wave a (new token, head), 64 keys at a time: a lane scores a key, the
// wave takes the running maximum and sum, then each lane gathers DIM / 64 of
// the output's columns over the keys.
template <int DIM>
__global__ __launch_bounds__(64) void attend_row_kernel(Attend a) {
  constexpr int C = DIM / 64;
  __shared__ float qs[DIM];
  const int64_t t = blockIdx.x;
  const int head = blockIdx.y, kvh = head / a.group, lane = threadIdx.x;
  int64_t lo = 0, hi = a.batch;  // the sequence of token t: starts[lo] <= t < starts[lo + 1]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  uint16_t* out = a.out + (t * a.heads + head) * DIM;
  float o[C] = {}, top = -INFINITY, sum = 0.0f;
  if (t >= a.starts[lo] && t < a.starts[lo + 1]) {
    const int64_t len = min(int64_t(a.seq_lens[lo]), a.table_keys);
    const int64_t pos = int64_t(a.seq_lens[lo]) - a.starts[lo + 1] + t;
    const int64_t end = a.causal ? min(len, pos + 1) : len;
    const int64_t begin = a.window > 0 ? max(pos - a.window + 1, int64_t(0)) : 0;
    const int32_t* table = a.table + lo * a.table_stride;
    for (int c = lane; c < DIM; c += 64)
      qs[c] = bf16_to_f32(a.q[t * a.q_token + head * a.q_head + c]);
    __syncthreads();
    for (int64_t j0 = begin; j0 < end; j0 += 64) {
      const int64_t j = j0 + lane;
      int64_t at = -1;
      float s = -INFINITY;
      if (j < end) {
        const int64_t page = table[j >> a.page_bits];
        if (page >= 0 && page < a.num_pages)
          at = ((page * a.kv_heads + kvh) << a.page_bits) + (j & ((1 << a.page_bits) - 1));
      }
      if (at >= 0) {
        float d = 0.0f;
        for (int c = 0; c < DIM; c += 4) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(a.k_codes + at * DIM + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) d += qs[c + i] * e4m3_to_f32(w >> (8 * i));
        }
        s = ldexpf(d, a.k_exps[at]) * a.scale;
      }
      const float m = fmaxf(top, wave_max(s));
      if (__ballot(at >= 0) == 0) continue;
      const float p = at >= 0 ? expf(s - m) : 0.0f;
      const float old = top == -INFINITY ? 0.0f : expf(top - m);
      float ps = p;
#pragma unroll
      for (int x = 32; x > 0; x >>= 1) ps += __shfl_xor(ps, x, 64);
      sum = sum * old + ps;
      top = m;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= old;
      const float pe = at >= 0 ? ldexpf(p, a.v_exps[at]) : 0.0f;
      for (int x = 0; x < 64; ++x) {
        const int64_t ax = __shfl(at, x, 64);
        if (ax < 0) continue;
        const float px = __shfl(pe, x, 64);
#pragma unroll
        for (int c = 0; c < C; ++c)
          o[c] += px * e4m3_to_f32(a.v_codes[ax * DIM + c * 64 + lane]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float v = sum == 0.0f ? 0.0f : o[c] / sum;
    out[c * 64 + lane] = f32_to_bf16_rne(v);
  }
}

}  // namespace

extern "C" {

int tcfp_kv_cache_write(const void* k, int64_t k_token_stride, int64_t k_head_stride,
                        const void* v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                        int64_t tokens, int kv_heads, int dim, const int64_t* slots,
                        int64_t num_pages, int page_size, uint8_t* k_codes, uint8_t* v_codes,
                        int8_t* k_exps, int8_t* v_exps, void* stream) {
  if (tokens < 0 || !cache_ok(num_pages, page_size, kv_heads, dim)) return TCFP_ERR_SHAPE;
  if (dtype != TCFP_DTYPE_F32 && dtype != TCFP_DTYPE_BF16) return TCFP_ERR_DTYPE;
  const int64_t unit = dtype == TCFP_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(v_codes) ||
      k_token_stride % unit || k_head_stride % unit || v_token_stride % unit ||
      v_head_stride % unit)
    return TCFP_ERR_ALIGN;
  if (tokens == 0 || num_pages == 0) return TCFP_OK;
  const Strided x{{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}};
  const Pool pool{{k_codes, v_codes}, {k_exps, v_exps}, num_pages * page_size, kv_heads,
                  log2i(page_size)};
  const auto st = static_cast<hipStream_t>(stream);
  const int64_t items = tokens * kv_heads, per = kThreads / (dim / 8);
  const int64_t blocks = (items + per - 1) / per;
  if (!grid_x_fits(blocks, kThreads)) return TCFP_ERR_SHAPE;
  const dim3 grid(unsigned(blocks), 2);
#define TCFP_KVW(T, D) cache_write_kernel<T, D><<<grid, kThreads, 0, st>>>(x, pool, slots, items)
#define TCFP_KVW_D(T)                    \
  do {                                   \
    if (dim == 64) TCFP_KVW(T, 64);      \
    else if (dim == 128) TCFP_KVW(T, 128); \
    else TCFP_KVW(T, 256);               \
  } while (0)
  if (dtype == TCFP_DTYPE_F32) TCFP_KVW_D(float); else TCFP_KVW_D(uint16_t);
#undef TCFP_KVW_D
#undef TCFP_KVW
  return launch_status();
}

int tcfp_kv_cache_read(const uint8_t* k_codes, const uint8_t* v_codes, const int8_t* k_exps,
                       const int8_t* v_exps, int64_t num_pages, int page_size, int kv_heads,
                       int dim, const int64_t* slots, int64_t tokens, void* k, void* v,
                       int dtype, void* stream) {
  if (tokens < 0 || !cache_ok(num_pages, page_size, kv_heads, dim)) return TCFP_ERR_SHAPE;
  if (dtype != TCFP_DTYPE_F32 && dtype != TCFP_DTYPE_BF16) return TCFP_ERR_DTYPE;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(v_codes))
    return TCFP_ERR_ALIGN;
  if (tokens == 0) return TCFP_OK;
  const Pool pool{{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(v_codes)},
                  {const_cast<int8_t*>(k_exps), const_cast<int8_t*>(v_exps)},
                  num_pages * page_size, kv_heads, log2i(page_size)};
  const auto st = static_cast<hipStream_t>(stream);
  const int64_t items = tokens * kv_heads, per = kThreads / (dim / 8);
  const int64_t blocks = (items + per - 1) / per;
  if (!grid_x_fits(blocks, kThreads)) return TCFP_ERR_SHAPE;
  const dim3 grid(unsigned(blocks), 2);
#define TCFP_KVR(T, D)                                                                 \
  cache_read_kernel<T, D><<<grid, kThreads, 0, st>>>(pool, slots, items,               \
                                                     static_cast<T*>(k), static_cast<T*>(v))
#define TCFP_KVR_D(T)                    \
  do {                                   \
    if (dim == 64) TCFP_KVR(T, 64);      \
    else if (dim == 128) TCFP_KVR(T, 128); \
    else TCFP_KVR(T, 256);               \
  } while (0)
  if (dtype == TCFP_DTYPE_F32) TCFP_KVR_D(float); else TCFP_KVR_D(uint16_t);
#undef TCFP_KVR_D
#undef TCFP_KVR
  return launch_status();
}

size_t tcfp_paged_attention_workspace_bytes(int64_t tokens, int heads, int kv_heads, int dim,
                                            int64_t batch, int64_t max_query_len,
                                            int64_t max_seq_len) {
  (void)tokens, (void)heads, (void)kv_heads, (void)dim, (void)batch;
  (void)max_query_len, (void)max_seq_len;
  return 0;
}

int tcfp_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                         const uint8_t* k_codes, const uint8_t* v_codes, const int8_t* k_exps,
                         const int8_t* v_exps, int64_t num_pages, int page_size, int kv_heads,
                         int dim, const int32_t* page_table, int64_t table_stride,
                         int64_t table_width, const int32_t* seq_lens,
                         const int32_t* query_start, int64_t batch, int64_t tokens, int heads,
                         int64_t max_query_len, int64_t max_seq_len, float scale, int causal,
                         int64_t window, void* out, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (tokens < 0 || batch < 0 || batch > 65535 || tokens > INT32_MAX ||
      !cache_ok(num_pages, page_size, kv_heads, dim))
    return TCFP_ERR_SHAPE;
  if (heads <= 0 || heads > 65535 || heads % kv_heads != 0) return TCFP_ERR_SHAPE;
  if (table_width < 0 || table_stride < table_width || max_query_len < 0 || max_seq_len < 0 ||
      window < 0)
    return TCFP_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_codes) || !aligned16(v_codes) ||
      q_token_stride % 8 || q_head_stride % 8)
    return TCFP_ERR_ALIGN;
  if (tokens == 0) return TCFP_OK;
  if (batch == 0) return TCFP_ERR_SHAPE;
  (void)workspace, (void)workspace_bytes;
  const Attend a{static_cast<const uint16_t*>(q), q_token_stride, q_head_stride, k_codes, v_codes,
                 k_exps, v_exps, num_pages, log2i(page_size), kv_heads, page_table, table_stride,
                 table_width * page_size, seq_lens, query_start, batch, tokens, heads,
                 heads / kv_heads, scale, causal, window, static_cast<uint16_t*>(out)};
  const auto st = static_cast<hipStream_t>(stream);
  if (!grid_x_fits(tokens, 64)) return TCFP_ERR_SHAPE;
  const dim3 grid{unsigned(tokens), unsigned(heads)};
  if (dim == 64) attend_row_kernel<64><<<grid, 64, 0, st>>>(a);
  else if (dim == 128) attend_row_kernel<128><<<grid, 64, 0, st>>>(a);
  else attend_row_kernel<256><<<grid, 64, 0, st>>>(a);
  return launch_status();
}

}  // extern "C"
