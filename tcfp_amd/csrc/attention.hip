// Paged K/V cache in E4M3 codes with one power-of-two exponent per token and
// head, and attention of new tokens over it, for gfx950.
//
//   codes [num_pages, kv_heads, page_size, dim], exps [num_pages, kv_heads,
//   page_size]: the keys of one page and head are one contiguous run, so a
//   tile of keys is read in whole lines whatever the number of heads.
#include <algorithm>
#include <cmath>

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

// DIM / 8 lanes a (token, head), 8 values each; blockIdx.y: K or V.  Bound by HBM:
// 8000 tokens of 8 heads of 128 in fp32 15.7 us (5.2 TB/s), 30011 tokens read
// into bf16 40.6 us (4.6 TB/s); 64 tokens 2.7 us, a launch and two latencies.
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
//
// The rows of a (sequence, K/V head) are its new tokens times the group of
// query heads that share the head: row r is token r / group, head r % group
// of the group.  A workgroup takes a tile of rows over a run of keys; rows whose
// keys are all in one run are finished there, the others leave (sum p v, max,
// sum p) for a joining launch, which adds the runs in order.
//
//   S^T = K Q^T      A = K codes, B = Q   keys down the registers, rows across lanes
//   O^T += V^T P^T   A = V^T,     B = P^T
// Transposed like this, a lane's S values are the P values that the second
// product wants of it (the order of its keys is the same permutation on both
// sides), a row's maximum and sum are over a lane's own registers and one or
// two other lanes, and rescaling O is a multiplication by the lane's own factor.
//
// The first product runs on the codes as they are cached: q = hi + lo in E4M3
// with one power-of-two scale a row is exact for bf16 values down to 2^-10 of
// the row's largest (4 + 4 significant bits) and within 2^-18 of the largest
// below that; the matrix instruction applies 2^e of a key as its block scale,
// and two FP8 products cost what one bf16 product would, without converting K.
// V is converted to bf16 with its exponent (both exact) and P is rounded to
// bf16: 2^-9 of a weight, where the result's own rounding to bf16 is 2^-9 too.
// Scores, maxima and sums are fp32; the sum is of P before its rounding.  But the
// FP8 instructions add the products of eight neighbouring columns with no bit under
// 2^-13 of the largest (what is further below it is lost; across such groups the
// sum is fp32's), so a score is off by some 2^-19, at most 2^-16 seen, of scale *
// sum |q k|: what a change of q by as much would do, where its rounding to bf16 was
// 2^-9 and the cache's K has 2^-4.  bf16 products would not lose them; their K takes
// twice the LDS and its reads, of which the prompts' kernels have none to spare.

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int kMaxSplits = 64;
constexpr int64_t kMostKeys = 1 << 30;  // positions stay clear of 2^31

struct Attend {
  const uint16_t* q;
  int64_t q_token, q_head;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const int8_t* k_exps;
  const int8_t* v_exps;
  int num_pages;
  int page_bits;
  int kv_heads;
  const int32_t* table;
  int64_t table_stride;
  int table_keys;  // keys that a row of the table spans
  const int32_t* seq_lens;
  const int32_t* starts;
  int batch;
  int tokens;
  int heads;
  int group;        // heads / kv_heads
  float c;          // |scale| * log2(e), 1 for a scale of 0
  float q_mul;      // sign of the scale
  int causal;
  int window;       // 0: none
  int tiles;        // row tiles of a (sequence, head) in the launch
  int splits;       // of a row tile's keys
  int chunk;        // keys of a split but the last
  int sets;         // (sequence, K/V head, split)s of the many-rows launches
  int tiles_first;  // their order on an XCD
  int workers;      // workgroups of the few-rows launch
  int whole;        // their items are not divided
  uint16_t* out;
  float* part;      // [splits][tokens * heads][dim]
  float* part_ml;   // [splits][tokens * heads][2]: max (in units of s), sum
};

// The rows of sequence b.
struct Seq {
  int start, new_tokens, len, pos0, rows;
};
TCFP_DEV Seq sequence(const Attend& a, int b) {
  Seq s;
  s.start = min(max(a.starts[b], 0), a.tokens);
  s.new_tokens = max(min(a.starts[b + 1], a.tokens) - s.start, 0);
  const int total = a.seq_lens[b];
  s.len = min(max(total, 0), a.table_keys);
  s.pos0 = total - s.new_tokens;  // position of the first new token
  s.rows = s.new_tokens * a.group;
  return s;
}
// Keys that new token i sees: [lo, hi).
TCFP_DEV int key_lo(const Attend& a, const Seq& s, int i) {
  return a.window > 0 ? max(s.pos0 + i - a.window + 1, 0) : 0;
}
TCFP_DEV int key_hi(const Attend& a, const Seq& s, int i) {
  return a.causal ? min(s.len, s.pos0 + i + 1) : s.len;
}
// Keys of a tile of rows [r0, r0 + n) and the splits that hold some.
struct Keys {
  int begin, end;  // begin is a multiple of 64
  int live;
};
TCFP_DEV Keys keys_of(const Attend& a, const Seq& s, int r0, int n) {
  Keys k;
  k.begin = key_lo(a, s, r0 / a.group) & ~63;
  k.end = key_hi(a, s, (min(r0 + n, s.rows) - 1) / a.group);
  const int span = max(k.end - k.begin, 0);
  k.live = min((span + a.chunk - 1) / a.chunk, a.splits);
  return k;
}

// A lane's N runs of 32 values of a row of q (p, p + step, ...) as E4M3 hi + lo,
// with one scale for the row, whose other values lanes +- 32 (LANES == 2) or
// +- 16, 32 (LANES == 4) hold; the scale is returned as the biased exponent that
// the matrix instructions take.  (Their scale of a lane belongs to a block of 32
// columns that is not the one whose values the lane holds: one scale for the
// row, and for K's row, leaves that without effect.)
template <int N, int LANES, int APART>
TCFP_DEV int split_q(const uint16_t* p, int step, float mul, v8i* hi, v8i* lo) {
  uint32_t m = 0;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      float v[8];
      load8(p + n * step + (i & 8) + (i >> 4) * APART, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = umax(m, absbits(v[j]));
    }
  if constexpr (LANES == 4) m = umax(m, uint32_t(__shfl_xor(int(m), 16, 64)));
  m = umax(m, uint32_t(__shfl_xor(int(m), 32, 64)));
  const int e = block_exponent(__uint_as_float(m), kE4M3Max);
  const float up = exp2i(-e) * mul;  // (no value passes 448 but where the row's scale is NaN)
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      float v[8];
      load8(p + n * step + (i & 8) + (i >> 4) * APART, v);
#pragma unroll
      for (int h = 0; h < 8; h += 4) {
        float x[4], r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = v[h + j] * up;
        const uint32_t w = cvt4_fp8<TCFP_FP8_E4M3>(x[0], x[1], x[2], x[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = x[j] - e4m3_to_f32(w >> (8 * j));
        hi[n][(i + h) / 4] = int(w);
        lo[n][(i + h) / 4] = int(cvt4_fp8<TCFP_FP8_E4M3>(r[0], r[1], r[2], r[3]));
      }
    }
  return e + 127;  // (255, the format's NaN, where the row holds an infinity)
}

// Two neighbouring codes (of bytes 0, 1 or 2, 3) times 2^e as bf16.
template <bool HIGH>
TCFP_DEV uint32_t deq2(uint32_t w, float scale) {
  const v2bf r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH);
  return __builtin_bit_cast(uint32_t, r);
}
// The low / high halves of two words, one after the other.
TCFP_DEV uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
TCFP_DEV uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// 2^e of the signed byte j of w, for the exponents that a cache is written with
// (-126 ... 120).
TCFP_DEV float exp_scale(uint32_t w, int j) {
  return __uint_as_float(uint32_t(max(int(int8_t(w >> (8 * j))) + 127, 0)) << 23);
}
// Bit 7 of the bytes of w that are NaN codes.
TCFP_DEV uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
// w with its NaN codes made zero.
TCFP_DEV uint32_t without_nan(uint32_t w) { return w & ~((nan_bytes(w) >> 7) * 255u); }
TCFP_DEV v8bf as_bf(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(v8bf, make_uint4(a, b, c, d));
}
TCFP_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

TCFP_DEV int valid_page(const Attend& a, int p) { return p >= 0 && p < a.num_pages ? p : -1; }

// NaN codes of V.  A row takes sum p v over all keys of a step, with p = 0 for the
// keys that it does not see, so a NaN must not stand in a step whose keys some row
// does not see (0 * NaN).  There it counts as zero, the step's keys are noted, and
// mark_nan makes the columns NaN afterwards, for the rows that see the key.  (A
// workgroup's notes, in LDS, are of all it does: a row's own bounds say which of
// their keys it sees.)
struct NanKeys {
  int begin, end;  // none: end <= begin
};
TCFP_DEV void note_nan(NanKeys* nans, int key0, int keys) {
  atomicMin(&nans->begin, key0);
  atomicMax(&nans->end, key0 + keys);
}
// Calls mark(w, nan_bytes) for the lane's words of V (word w is codes w * STRIDE + at
// ...) that hold a NaN of a key in [n.begin, n.end) and [lo, hi), one key after
// another: a cache that holds NaN is no case to be fast at.
template <int D, int WORDS, int STRIDE, typename Mark>
TCFP_DEV void mark_nan(const Attend& a, const int32_t* table, int kvh, NanKeys n, int lo, int hi,
                       int at, Mark mark) {
  const int end = min(n.end, hi);
#pragma unroll 1
  for (int key = max(n.begin, lo); key < end; ++key) {
    const int page = valid_page(a, table[key >> a.page_bits]);
    if (page < 0) continue;
    const uint8_t* v = a.v_codes +
                       ((((int64_t(page) * a.kv_heads + kvh) << a.page_bits) +
                         (key & ((1 << a.page_bits) - 1))) * D + at);
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(v + w * STRIDE);
      if (nan_bytes(x)) mark(w, nan_bytes(x));
    }
  }
}
TCFP_DEV bool byte_of(uint32_t nans, int byte) { return (nans >> (8 * byte + 7)) & 1u; }

// Rows of q before the first (lead) and from behind the last sequence (tail):
// zeros, for `heads` heads from head `first`.
TCFP_DEV void zero_rest(const Attend& a, int lead, int tail, int first, int heads, int dim) {
  const int words = heads * dim / 2, rest = max(a.tokens - max(tail, lead), 0);
  for (int i = 0; i < lead + rest; ++i) {
    const int t = i < lead ? i : max(tail, lead) + i - lead;
    uint32_t* p = reinterpret_cast<uint32_t*>(a.out + (int64_t(t) * a.heads + first) * dim);
    for (int x = threadIdx.x; x < words; x += blockDim.x) p[x] = 0;
  }
}

// ---- few rows: one token a sequence, a few drafts ----------------------------
//
// Bound by reading the cache: 64 sequences of up to 8192 tokens, 32 / 8 heads of
// 128, 132 us with the joining launch (5.26 TB/s of codes and exponents), heads
// of 64 75 us, heads of 256 (16 / 8) 248 us (5.6 TB/s); one sequence of 127
// tokens 5.3 us, a chain of latencies: lengths, page table, keys, the waves'
// join.  A wave takes KT keys at a time straight into registers, the next KT in
// flight; nothing of K or V passes through LDS.  The four waves of a workgroup
// take turns over its run of keys and are joined at its end.
template <int D>
struct FewShape {
  static constexpr int KT = 32;                  // keys of a wave's step
  static constexpr int KG = KT / 16;             // groups of 16 keys, each in one page
  static constexpr int DS = D == 256 ? 2 : 1;    // 128-column steps of the first product
  static constexpr int VW = D / 64;              // words of a lane's share of a V row
  static constexpr int NI = D / 16;              // column tiles of the output
};

template <int D>
struct FewTile {
  using S = FewShape<D>;
  uint4 k[S::KG][S::DS][2];
  uint32_t v[S::KG][4][S::VW];
  int ke[S::KG];
  uint32_t ve[S::KG];
  int page[S::KG];
};

constexpr int kSegKeys = 2048;  // keys whose pages are held in LDS at a time

// A value that is the same in every lane, as the wave's own.
TCFP_DEV int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
TCFP_DEV int64_t scalar(int64_t v) {
  return int64_t(uint64_t(uint32_t(scalar(int(uint64_t(v) >> 32)))) << 32 |
                 uint32_t(scalar(int(uint32_t(uint64_t(v))))));
}

template <int N>
TCFP_DEV void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    w[0] = t.x; w[1] = t.y;
  } else {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
  }
}
// Lane offsets of a group of 16 keys: its share of a key of K, of four keys of
// V, of their exponents.
struct FewLane {
  uint32_t k, v, ke, ve;
};
template <int D>
TCFP_DEV FewLane few_lane(int lane) {
  const uint32_t col = lane & 15, g4 = lane >> 4;
  return {col * D + (D == 64 ? (g4 & 1) * 16 : g4 * 16), 4 * g4 * D + col * (D / 16), col, 4 * g4};
}

template <int D>
TCFP_DEV void few_load(const Attend& a, int kvh, const int* pages, int seg, int seg_end,
                       int key0, const FewLane& off, FewTile<D>& t) {
  using S = FewShape<D>;
#pragma unroll
  for (int g = 0; g < S::KG; ++g) {
    const int key = key0 + 16 * g;
    // (past the end: the last page's entry, masked)
    const int held = scalar(pages[(min(key, seg_end - 1) >> a.page_bits) - (seg >> a.page_bits)]);
    t.page[g] = key < seg_end ? held : -1;
    // (a missing page is read from page 0 -- the pool has pages -- and masked)
    const int64_t at = ((int64_t(max(held, 0)) * a.kv_heads + kvh) << a.page_bits) +
                       (key & ((1 << a.page_bits) - 1));
    const uint8_t* kp = a.k_codes + at * D;
#pragma unroll
    for (int s = 0; s < S::DS; ++s) {
      t.k[g][s][0] = *reinterpret_cast<const uint4*>(kp + off.k + s * 128);
      t.k[g][s][1] = *reinterpret_cast<const uint4*>(kp + off.k + s * 128 + (D == 64 ? 32 : 64));
    }
    t.ke[g] = (a.k_exps + at)[off.ke];
    const uint8_t* vp = a.v_codes + at * D;
#pragma unroll
    for (int r = 0; r < 4; ++r) load_words<S::VW>(vp + off.v + r * D, t.v[g][r]);
    t.ve[g] = *reinterpret_cast<const uint32_t*>(a.v_exps + at + off.ve);
  }
}

template <int D, int NT>
struct FewState {
  using S = FewShape<D>;
  v8i qhi[NT][S::DS], qlo[NT][S::DS];  // D == 64: hi and lo side by side in qhi
  int qe[NT];
  int lo[NT], hi[NT];                  // keys that the lane's row sees
  float m[NT], l[NT];
  v4f o[NT][S::NI];
};

// One step over KT keys; masked: some row does not see all of them (or a page
// is missing).  [all_lo, all_hi): keys that any row sees.
template <int D, int NT, bool masked>
TCFP_DEV void few_step(const Attend& a, FewState<D, NT>& st, FewTile<D>& t, int key0,
                       int all_lo, int all_hi, NanKeys* nans) {
  using S = FewShape<D>;
  const int lane = threadIdx.x & 63, g4 = lane >> 4;
  bool nan = false;
  if (masked) {
#pragma unroll
    for (int g = 0; g < S::KG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = key0 + 16 * g + 4 * g4 + r;
        const bool dead = key < all_lo || key >= all_hi || t.page[g] < 0;
        // what no row sees counts as zero, whatever the page holds there
        uint32_t codes = 0;
#pragma unroll
        for (int w = 0; w < S::VW; ++w) {
          if (dead) t.v[g][r][w] = 0;
          codes |= nan_bytes(t.v[g][r][w]);
          t.v[g][r][w] = without_nan(t.v[g][r][w]);
        }
        nan |= codes != 0;
        if (dead) t.ve[g] &= ~(0xFFu << (8 * r));
      }
  }
  float p[NT][S::KG][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < S::KG; ++g) {
      v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int d = 0; d < S::DS; ++d) {
        v8i k;
        k[0] = int(t.k[g][d][0].x); k[1] = int(t.k[g][d][0].y);
        k[2] = int(t.k[g][d][0].z); k[3] = int(t.k[g][d][0].w);
        k[4] = int(t.k[g][d][1].x); k[5] = int(t.k[g][d][1].y);
        k[6] = int(t.k[g][d][1].z); k[7] = int(t.k[g][d][1].w);
        s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, st.qhi[n][d], s, 0, 0, 0,
                                                             t.ke[g] + 127, 0, st.qe[n]);
        if constexpr (D != 64)
          s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, st.qlo[n][d], s, 0, 0, 0,
                                                               t.ke[g] + 127, 0, st.qe[n]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) p[n][g][r] = s[r];
    }
    if (masked) {
#pragma unroll
      for (int g = 0; g < S::KG; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + 16 * g + 4 * g4 + r;
          if (key < st.lo[n] || key >= st.hi[n] || t.page[g] < 0) p[n][g][r] = -INFINITY;
        }
    }
#pragma unroll
    for (int g = 0; g < S::KG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, p[n][g][r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    top = fmaxf(top, st.m[n]);
    if (__ballot(top > st.m[n])) {
      const float f = top == st.m[n] ? 1.0f : exp2_fast((st.m[n] - top) * a.c);
      st.m[n] = top;
      st.l[n] *= f;
#pragma unroll
      for (int i = 0; i < S::NI; ++i) st.o[n][i] *= f;
    }
    const float off = top == -INFINITY ? 0.0f : top * a.c;
#pragma unroll
    for (int g = 0; g < S::KG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[n][g][r] = exp2_fast(__builtin_fmaf(p[n][g][r], a.c, -off));
        st.l[n] += p[n][g][r];
      }
  }
#pragma unroll
  for (int g = 0; g < S::KG; g += 2) {  // 32 keys of the second product
    v8bf pf[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      pf[n] = as_bf(pack_bf16(p[n][g][0], p[n][g][1]), pack_bf16(p[n][g][2], p[n][g][3]),
                    pack_bf16(p[n][g + 1][0], p[n][g + 1][1]),
                    pack_bf16(p[n][g + 1][2], p[n][g + 1][3]));
    float sc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sc[j] = exp_scale(t.ve[g + j / 4], j % 4);
#pragma unroll
    for (int w = 0; w < S::VW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // two columns of the lane's share at a time
        uint32_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] = h ? deq2<true>(t.v[g + j / 4][j % 4][w], sc[j])
                   : deq2<false>(t.v[g + j / 4][j % 4][w], sc[j]);
        const v8bf v0 = as_bf(lows(x[0], x[1]), lows(x[2], x[3]), lows(x[4], x[5]), lows(x[6], x[7]));
        const v8bf v1 =
            as_bf(highs(x[0], x[1]), highs(x[2], x[3]), highs(x[4], x[5]), highs(x[6], x[7]));
        const int i = 4 * w + 2 * h;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          st.o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pf[n], st.o[n][i], 0, 0, 0);
          st.o[n][i + 1] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pf[n], st.o[n][i + 1], 0, 0, 0);
        }
      }
  }
  if (masked && nan) note_nan(nans, key0, S::KT);
}

// The value of a lane (its number the same in every lane).
TCFP_DEV int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
TCFP_DEV int64_t of_lane(int64_t v, int lane) {
  return int64_t(uint64_t(uint32_t(of_lane(int(uint64_t(v) >> 32), lane))) << 32 |
                 uint32_t(of_lane(int(uint32_t(uint64_t(v))), lane)));
}

// The few-rows launch cuts the batch's keys into equal runs, whatever the
// lengths: an item is a (sequence, row tile, head), its keys count in units of
// kUnit, and workgroup w takes the units [w q, (w + 1) q) of all items in order
// (q from the lengths, which are on the device: every workgroup adds them up).
// An item within one workgroup is finished there; of the others each part goes
// to a place of its own, 2 w for a workgroup's first part and 2 w + 1 for an item
// that only starts in it, and the joining launch adds an item's parts in order.
// With `whole` an item is one unit and nothing is joined.
constexpr int kUnit = 128;

// Items of sequence b: units of each, and how many there are.
TCFP_DEV int units_of(const Attend& a, const Seq& s) {
  if (a.whole) return 1;
  const int begin = key_lo(a, s, 0) & ~63, end = key_hi(a, s, s.new_tokens - 1);
  return max((end - begin + kUnit - 1) / kUnit, 1);
}
TCFP_DEV int items_of(const Attend& a, const Seq& s, int tile_rows) {
  return (s.rows + tile_rows - 1) / tile_rows * a.kv_heads;
}

// a / b of non-negative numbers, by the 32-bit division where that does.
TCFP_DEV int64_t divide(int64_t a, int64_t b) {
  if (uint64_t(a | b) >> 32) return a / b;
  return uint32_t(a) / uint32_t(b);
}

// Units of a workgroup of the launch: two at least, as a part costs a quarter of
// the time of its keys.
TCFP_DEV int64_t share_of(const Attend& a, int64_t total) {
  return max(divide(total + a.workers - 1, a.workers), int64_t(a.whole ? 1 : 2));
}

// A sequence, the units before it and those of the whole batch.
struct Found {
  int b;
  Seq seq;
  int64_t before, total;
  int lead, tail;  // rows of q before the first sequence, and up to the last one's end
};
struct FindLds {
  int64_t wave[4], before;
  Seq seq;
  int b;
};

// The sequence for which pick(seq, units before it, its units, all units) holds
// -- for one at most -- sought by a workgroup of 256 with 256 sequences at a
// time, or by each wave for itself where there are at most 64; false: none.
template <typename Pick>
TCFP_DEV bool find(const Attend& a, int tile_rows, FindLds& lds, Pick pick, Found& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (a.batch == 1) {
    f.seq = sequence(a, 0);
    const int64_t n =
        f.seq.rows > 0 ? int64_t(units_of(a, f.seq)) * items_of(a, f.seq, tile_rows) : 0;
    f.b = 0;
    f.before = 0;
    f.total = n;
    f.lead = f.seq.start;
    f.tail = f.seq.start + f.seq.new_tokens;
    return pick(f.seq, 0, n, n);
  }
  if (a.batch <= 64) {
    Seq s{};
    int64_t n = 0;
    if (lane < a.batch) {
      s = sequence(a, lane);
      if (s.rows > 0) n = int64_t(units_of(a, s)) * items_of(a, s, tile_rows);
    }
    int64_t upto = n;
    for (int x = 1; x < a.batch; x <<= 1) {
      const int64_t y = __shfl_up(upto, x, 64);
      if (lane >= x) upto += y;
    }
    f.total = of_lane(upto, a.batch - 1);
    f.lead = scalar(s.start);  // (of the first lane)
    f.tail = of_lane(s.start + s.new_tokens, a.batch - 1);
    const uint64_t here = __ballot(lane < a.batch && pick(s, upto - n, n, f.total));
    if (!here) return false;
    f.b = __builtin_ctzll(here);
    f.before = of_lane(upto - n, f.b);
    f.seq = {of_lane(s.start, f.b), of_lane(s.new_tokens, f.b), of_lane(s.len, f.b),
             of_lane(s.pos0, f.b), of_lane(s.rows, f.b)};
    return true;
  }
  Seq s{};
  int64_t n = 0, upto = 0, chunk = 0;  // units of the thread's sequence, of the wave's up to it, of the 256
  auto scan = [&](int b0) {
    const int b = b0 + int(threadIdx.x);
    s = Seq{};
    n = 0;
    if (b < a.batch) {
      s = sequence(a, b);
      if (s.rows > 0) n = int64_t(units_of(a, s)) * items_of(a, s, tile_rows);
    }
    upto = n;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int64_t y = __shfl_up(upto, x, 64);
      if (lane >= x) upto += y;
    }
    if (lane == 63) lds.wave[wave] = upto;
    __syncthreads();
    chunk = lds.wave[0] + lds.wave[1] + lds.wave[2] + lds.wave[3];
    for (int w = 0; w < wave; ++w) upto += lds.wave[w];
    __syncthreads();
  };
  const Seq end = sequence(a, a.batch - 1);
  f.lead = sequence(a, 0).start;
  f.tail = end.start + end.new_tokens;
  f.total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 256) {
    scan(b0);
    f.total += chunk;
  }
  f.total = scalar(f.total);
  int64_t start = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 256) {
    if (a.batch > 256) scan(b0);
    const bool here = b0 + int(threadIdx.x) < a.batch && pick(s, start + upto - n, n, f.total);
    if (here) {
      lds.b = b0 + int(threadIdx.x);
      lds.seq = s;
      lds.before = start + upto - n;
    }
    if (__syncthreads_or(here)) {
      f.b = scalar(lds.b);
      f.before = scalar(lds.before);
      f.seq = {scalar(lds.seq.start), scalar(lds.seq.new_tokens), scalar(lds.seq.len),
               scalar(lds.seq.pos0), scalar(lds.seq.rows)};
      return true;
    }
    start += chunk;
  }
  return false;
}

template <int D, int NT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_few_kernel(Attend a) {
  using S = FewShape<D>;
  constexpr int RT = 16 * NT;
  __shared__ int pages[kSegKeys / 16];
  __shared__ float ml[4][RT][2];
  __shared__ float4 xo[4][8][64];
  __shared__ FindLds fl;
  __shared__ NanKeys nans;
  if (threadIdx.x == 0) nans = {INT32_MAX, 0};  // (a barrier follows before any step)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g4 = lane >> 4;
  const FewLane off = few_lane<D>(lane);
  Found f;
  const bool any = find(
      a, RT, fl,
      [&](const Seq&, int64_t first, int64_t n, int64_t total) {
        const int64_t u = int64_t(blockIdx.x) * share_of(a, total);
        return n > 0 && u >= first && u < first + n;
      },
      f);
  if (blockIdx.x == 0) zero_rest(a, f.lead, f.tail, 0, a.heads, D);
  if (!any) return;
  const int64_t share = share_of(a, f.total);
  int64_t u = int64_t(blockIdx.x) * share, before = f.before;
  const int64_t u1 = min(u + share, f.total);
  int b = f.b;
  Seq seq = f.seq;
  while (u < u1) {
    const int units = units_of(a, seq), items = items_of(a, seq, RT);
    if (seq.rows <= 0 || u - before >= int64_t(units) * items) {  // on to the next sequence
      if (seq.rows > 0) before += int64_t(units) * items;
      seq = sequence(a, ++b);
      continue;
    }
    const int item = int(divide(u - before, units)), part = int(u - before - int64_t(item) * units);
    const int count = int(min(int64_t(units - part), u1 - u));
    const bool all = count == units;
    const int64_t place = 2 * int64_t(blockIdx.x) + (part == 0 ? 1 : 0);
    u += count;
    const int kvh = item % a.kv_heads, r0 = item / a.kv_heads * RT;
    const int32_t* table = a.table + int64_t(b) * a.table_stride;
    const int first = key_lo(a, seq, 0) & ~63, end = key_hi(a, seq, seq.new_tokens - 1);
    const int k0 = first + part * kUnit;
    const int k1 = a.whole ? end : min(end, k0 + count * kUnit);
    // (the first pages, on their way while q is split)
    const int page0 = k0 >> a.page_bits;
    int held = -1;
    if (k0 < k1 && page0 + int(threadIdx.x) <= (min(k1, k0 + kSegKeys) - 1) >> a.page_bits)
      held = table[page0 + threadIdx.x];
    FewState<D, NT> st;
    int lo_max = 0, hi_min = INT32_MAX;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(r0 + 16 * n + col, seq.rows - 1), i = r / a.group, h = r - i * a.group;
      const uint16_t* q = a.q + int64_t(seq.start + i) * a.q_token +
                          int64_t(kvh * a.group + h) * a.q_head;
      st.qe[n] = split_q<S::DS, 4, D == 64 ? 32 : 64>(q + (D == 64 ? (g4 & 1) * 16 : g4 * 16), 128, a.q_mul,
                                   st.qhi[n], st.qlo[n]);
      if (D == 64 && g4 >= 2) st.qhi[n][0] = st.qlo[n][0];
      st.lo[n] = key_lo(a, seq, i);
      st.hi[n] = key_hi(a, seq, i);
      st.m[n] = -INFINITY;
      st.l[n] = 0.0f;
#pragma unroll
      for (int x = 0; x < S::NI; ++x) st.o[n][x] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int last = min(r0 + RT, seq.rows) - 1;
    lo_max = key_lo(a, seq, last / a.group);
    hi_min = key_hi(a, seq, r0 / a.group);
    const int all_lo = key_lo(a, seq, r0 / a.group), all_hi = key_hi(a, seq, last / a.group);
    for (int seg = k0; seg < k1; seg += kSegKeys) {
      const int seg_end = min(seg + kSegKeys, k1);
      __syncthreads();
      {
        const int page = (seg >> a.page_bits) + int(threadIdx.x);
        if (page <= (seg_end - 1) >> a.page_bits)  // (128 at most)
          pages[threadIdx.x] = valid_page(a, seg == k0 ? held : table[page]);
      }
      __syncthreads();
      int key = seg + wave * S::KT;
      if (key >= seg_end) continue;  // (barriers: at the top of the loop only)
      FewTile<D> cur, nxt;
      few_load<D>(a, kvh, pages, seg, seg_end, key, off, cur);
      for (; key < seg_end; key += 4 * S::KT) {
        // (the last step loads its own keys again, from L2)
        const int next = key + 4 * S::KT < seg_end ? key + 4 * S::KT : key;
        few_load<D>(a, kvh, pages, seg, seg_end, next, off, nxt);
        bool hole = false;
#pragma unroll
        for (int g = 0; g < S::KG; ++g) hole |= cur.page[g] < 0;
        if (hole || key < lo_max || key + S::KT > hi_min)
          few_step<D, NT, true>(a, st, cur, key, all_lo, all_hi, &nans);
        else
          few_step<D, NT, false>(a, st, cur, key, all_lo, all_hi, &nans);
        cur = nxt;
      }
    }
    // ---- the four waves joined ----
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float l = st.l[n];
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      if (g4 == 0) {
        ml[wave][16 * n + col][0] = st.m[n];
        ml[wave][16 * n + col][1] = l;
      }
    }
    __syncthreads();
    if (nans.begin < nans.end) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
        mark_nan<D, 4 * S::VW, 4>(a, table, kvh, nans, st.lo[n], st.hi[n], 4 * g4 * (D / 16),
                                  [&](int w, uint32_t x) {
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                      if (byte_of(x, j))
                                        st.o[n][4 * (w % S::VW) + j][w / S::VW] = NAN;
                                  });
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][16 * n + col][0]);
      const float f = st.m[n] == top ? 1.0f : exp2_fast((st.m[n] - top) * a.c);
#pragma unroll
      for (int i0 = 0; i0 < S::NI; i0 += 8) {
        constexpr int IB = S::NI < 8 ? S::NI : 8;
#pragma unroll
        for (int i = 0; i < IB; ++i) {
          const v4f o = st.o[n][i0 + i] * f;
          xo[wave][i][lane] = make_float4(o[0], o[1], o[2], o[3]);
        }
        __syncthreads();
        // thread: columns i0 + 2 i2, + 1 of a lane's four rows of O^T
        const int i2 = threadIdx.x >> 6;
        if (2 * i2 < IB) {
          float s[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float4 t = xo[0][2 * i2 + j][lane];
#pragma unroll
            for (int w = 1; w < 4; ++w) {
              const float4 u = xo[w][2 * i2 + j][lane];
              t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
            }
            s[j][0] = t.x; s[j][1] = t.y; s[j][2] = t.z; s[j][3] = t.w;
          }
          float lsum = 0.0f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float mw = ml[w][16 * n + col][0];
            lsum += ml[w][16 * n + col][1] *
                    (mw == top ? 1.0f : exp2_fast((mw - top) * a.c));
          }
          const int r = r0 + 16 * n + col;
          if (r < seq.rows) {
            const int i = r / a.group, h = r - i * a.group;
            const int64_t row = int64_t(seq.start + i) * a.heads + kvh * a.group + h;
            if (all) {
              const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
              for (int x = 0; x < 4; ++x)
                *reinterpret_cast<uint32_t*>(a.out + row * D + (4 * g4 + x) * (D / 16) + i0 +
                                             2 * i2) = pack_bf16(s[0][x] * inv, s[1][x] * inv);
            } else {
              const int64_t at = place * RT + 16 * n + col;
#pragma unroll
              for (int x = 0; x < 4; ++x)
                *reinterpret_cast<float2*>(a.part + at * D + (4 * g4 + x) * (D / 16) + i0 +
                                           2 * i2) = make_float2(s[0][x], s[1][x]);
              if (i0 == 0 && i2 == 0 && g4 == 0) {
                a.part_ml[2 * at] = top;
                a.part_ml[2 * at + 1] = lsum;
              }
            }
          }
        }
        __syncthreads();
      }
    }
  }
}

// Workgroups go round the 8 XCDs in turn.  The row tiles of a (sequence, head,
// split) read the same keys: they go to one XCD, whose L2 then serves them, the
// last tiles, which see the most keys, first; where there are fewer than eight
// such sets their tiles are dealt over all XCDs.  An XCD takes one set after the
// other, or, where its L2 holds the keys of all its sets, the last tiles of all of
// them first (ragged prompts of up to 1000 tokens, 16 heads of 64: 46.8 -> 33.5 us).
// False: nothing to do.
TCFP_DEV bool place(const Attend& a, int& tile, int& split, int& kvh, int& b) {
  const uint32_t tiles = uint32_t(a.tiles);
  uint32_t set, t;
  if (a.sets >= 8) {
    const uint32_t nth = blockIdx.x / 8, sets = (uint32_t(a.sets) + 7) / 8;
    t = a.tiles_first ? nth / sets : nth % tiles;
    // (in turn, from another one each time: an XCD deals its workgroups over its
    // four shader engines in turn too, and a long sequence would keep to one)
    set = (a.tiles_first ? (nth + t) % sets : nth / tiles) * 8 + blockIdx.x % 8;
  } else {
    set = blockIdx.x / tiles;
    t = blockIdx.x % tiles;
  }
  if (set >= uint32_t(a.sets)) return false;
  tile = a.tiles - 1 - int(t);
  split = int(set % uint32_t(a.splits));
  set /= uint32_t(a.splits);
  kvh = int(set % uint32_t(a.kv_heads));
  b = int(set / uint32_t(a.kv_heads));
  return true;
}

// ---- many rows: prompts ------------------------------------------------------
//
// Bound by the matrix and vector units together and by what passes between
// them.  (A 2048-token chunk over 14336 tokens, 32 / 8 heads of 128, which the
// eight-wave kernel takes, ran 553 us here, 485 with the exponentials taken out, 532
// without its second product, 414 without moving keys.)  One prompt of 2048 tokens,
// 32 / 8 heads of 128: 67 us; six ragged ones of up to 1000, 16 heads of 64: 30 us,
// vector units 56% and matrix units 16% busy.  A workgroup's four waves hold 32 rows
// each;
// per 64 keys K goes to LDS as codes and V as bf16, transposed and in the order
// of keys that P has in its registers (both buffered twice, the next 64 keys
// loaded into registers meanwhile), so every operand is read with 16-byte LDS
// reads.  16-byte chunks of a line are permuted by the row, which spreads eight
// rows' reads over the banks.
//
// KS == 2, for heads of 256: 64 rows a workgroup, two waves with half of a step's
// keys each, their sums joined at the end.  A step of these heads takes a wave
// alone on its SIMD 3.3 us; short prompts are as slow as their longest tile.
constexpr int kManyRows = 128, kManyKeys = 64;

template <int D>
struct ManyShape {
  static constexpr int DW = D / 64;            // words of a thread's share of a row
  static constexpr int KB = kManyKeys * D;     // bytes of K
  static constexpr int VB = kManyKeys * D * 2; // bytes of V
  static constexpr int BUF = KB + VB + 64;     // and 64 scale bytes
  static constexpr int DS = D / 64;            // 64-column steps of the first product
  static constexpr int DT = D / 32;            // 32-row tiles of O^T
};

// byte offset of 16-byte chunk c of K row `row`
template <int D>
TCFP_DEV int k_at(int row, int c) {
  if constexpr (D == 64) return row * D + ((c ^ ((row >> 1) & 3)) << 4);
  else return row * D + ((c ^ (row & 7)) << 4);
}
// and of V^T row (column of V) d: 8 chunks of 8 keys
TCFP_DEV int v_at(int d, int c) { return d * 128 + ((c ^ ((d ^ (d >> 3) ^ (d >> 6)) & 7)) << 4); }

template <int D>
struct ManyLoad {
  uint32_t k[4][ManyShape<D>::DW], v[4][ManyShape<D>::DW];
  uint32_t ke, ve;
  int page;
};

template <int N>
TCFP_DEV void store_lds(uint8_t* p, const uint32_t* w) {
  if constexpr (N == 1) *reinterpret_cast<uint32_t*>(p) = w[0];
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Thread: keys 4 kg ... 4 kg + 3 of the 64, bytes dg * D / 16 ... of their rows.
template <int D>
TCFP_DEV void many_load(const Attend& a, int kvh, int key0, int page, ManyLoad<D>& t) {
  const int kg = threadIdx.x >> 4, dg = threadIdx.x & 15;
  const int key = key0 + 4 * kg;
  page = valid_page(a, page);
  t.page = page;
  const int64_t at = ((int64_t(max(page, 0)) * a.kv_heads + kvh) << a.page_bits) +
                     (key & ((1 << a.page_bits) - 1));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    load_words<ManyShape<D>::DW>(a.k_codes + (at + j) * D + dg * (D / 16), t.k[j]);
    load_words<ManyShape<D>::DW>(a.v_codes + (at + j) * D + dg * (D / 16), t.v[j]);
  }
  t.ke = *reinterpret_cast<const uint32_t*>(a.k_exps + at);
  t.ve = *reinterpret_cast<const uint32_t*>(a.v_exps + at);
}

// The loaded keys into a buffer.  masked: some row of the workgroup does not
// see all of them; what no row sees counts as zero, and so does a NaN among the
// codes of V, which is noted.
template <int D>
TCFP_DEV void many_store(uint8_t* buf, ManyLoad<D>& t, int key0, bool masked, int all_lo,
                         int all_hi, NanKeys* nans) {
  using S = ManyShape<D>;
  const int kg = threadIdx.x >> 4, dg = threadIdx.x & 15;
  // 127 added to each byte
  uint32_t scales = ((t.ke & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) ^ (t.ke & 0x80808080u);
  if (masked) {
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = key0 + 4 * kg + j;
      const bool dead = key < all_lo || key >= all_hi || t.page < 0;
#pragma unroll
      for (int w = 0; w < S::DW; ++w) {
        if (dead) t.v[j][w] = 0;
        nan |= nan_bytes(t.v[j][w]) != 0;
        t.v[j][w] = without_nan(t.v[j][w]);
      }
      if (dead) t.ve &= ~(0xFFu << (8 * j));
    }
    if (nan) note_nan(nans, key0, kManyKeys);
    if (t.page < 0) scales = 0;  // no page: nobody sees these four keys
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int byte = dg * (D / 16);
    store_lds<S::DW>(buf + k_at<D>(4 * kg + j, byte >> 4) + (byte & 15), t.k[j]);
  }
  uint8_t* vt = buf + S::KB;
  const int c = (kg >> 2) * 2 + (kg & 1), sub = ((kg >> 1) & 1) * 8;
  float sc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sc[j] = exp_scale(t.ve, j);
#pragma unroll
  for (int w = 0; w < S::DW; ++w)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = h ? deq2<true>(t.v[j][w], sc[j]) : deq2<false>(t.v[j][w], sc[j]);
      const int d = dg * (D / 16) + 4 * w + 2 * h;
      *reinterpret_cast<uint2*>(vt + v_at(d, c) + sub) =
          make_uint2(lows(x[0], x[1]), lows(x[2], x[3]));
      *reinterpret_cast<uint2*>(vt + v_at(d + 1, c) + sub) =
          make_uint2(highs(x[0], x[1]), highs(x[2], x[3]));
    }
  if (dg == 0) *reinterpret_cast<uint32_t*>(buf + S::KB + S::VB + 4 * kg) = scales;
}

TCFP_DEV float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return (threadIdx.x & 32) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}

// The rows' sums over the keys of the upper half of a workgroup's waves, of which
// RW hold a row each, added to those of the lower half, through LDS.
template <int DT, int RW, int BYTES>
TCFP_DEV void join_halves(const Attend& a, uint8_t* lds, int wave, int lane, v16f* o, float& m,
                          float& l) {
  constexpr int N = 16 * DT;
  static_assert(RW * (N + 2) * 64 * 4 <= BYTES, "the sums fit where the keys were");
  float* const x = reinterpret_cast<float*>(lds) + wave % RW * (N + 2) * 64 + lane;
  if (wave >= RW) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[64 * i] = o[i / 16][i % 16];
    x[64 * N] = m;
    x[64 * N + 64] = l;
  }
  __syncthreads();
  if (wave < RW) {
    const float om = x[64 * N], top = fmaxf(m, om);
    const float f = m == top ? 1.0f : exp2_fast((m - top) * a.c);
    const float g = om == top ? 1.0f : exp2_fast((om - top) * a.c);
    m = top;
    l = l * f + x[64 * N + 64] * g;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i / 16][i % 16] = o[i / 16][i % 16] * f + x[64 * i] * g;
  }
  __syncthreads();
}

// mark_nan for a lane's columns of O^T, 8 g + 4 half ... of every 32.
template <int D>
TCFP_DEV void mark_nan_rows(const Attend& a, const int32_t* table, int kvh, const NanKeys& nans,
                            int lo, int hi, int half, v16f* o) {
  if (nans.begin >= nans.end) return;
  mark_nan<D, D / 8, 8>(a, table, kvh, nans, lo, hi, 4 * half, [&](int w, uint32_t x) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (byte_of(x, r)) o[w / 4][4 * (w % 4) + r] = NAN;
  });
}

template <int D, int KS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_many_kernel(Attend a) {
  using S = ManyShape<D>;
  constexpr int RT = kManyRows / KS, KT = 2 / KS;  // rows, and a wave's 32-key tiles of a step
  __shared__ uint4 lds4[2 * S::BUF / 16];
  __shared__ NanKeys nans;
  if (threadIdx.x == 0) nans = {INT32_MAX, 0};  // (a barrier follows before any step)
  uint8_t* const lds = reinterpret_cast<uint8_t*>(lds4);
  const int lane = threadIdx.x & 63, wave = scalar(int(threadIdx.x >> 6)), col = lane & 31, half = lane >> 5;
  int tile, split, kvh, b;
  if (!place(a, tile, split, kvh, b)) return;
  const Seq seq = sequence(a, b);
  if (split == 0 && tile == 0)
    zero_rest(a, b == 0 ? seq.start : 0,
              b == a.batch - 1 ? seq.start + seq.new_tokens : a.tokens, kvh * a.group, a.group, D);
  const int32_t* table = a.table + int64_t(b) * a.table_stride;
  const int kg = threadIdx.x >> 4;
  const int mine = wave % (4 / KS), kfirst = KS == 1 ? 0 : wave / 2;
  for (int r0 = tile * RT; r0 < seq.rows; r0 += a.tiles * RT) {
    const Keys keys = keys_of(a, seq, r0, RT);
    if (split >= max(keys.live, 1)) continue;
    const int k0 = keys.begin + split * a.chunk;
    const int k1 = split == a.splits - 1 ? keys.end : min(keys.end, k0 + a.chunk);
    // rows of the tile, of the wave and of the lane; rows past the last repeat it
    const int last = min(r0 + RT, seq.rows) - 1;
    const int row = min(r0 + 32 * mine + col, last), tok = row / a.group,
              head = row - tok * a.group;
    const int lo = key_lo(a, seq, tok), hi = key_hi(a, seq, tok);
    const int wfirst = min(r0 + 32 * mine, last) / a.group,
              wlast = min(r0 + 32 * mine + 31, last) / a.group;
    const int all_lo = key_lo(a, seq, r0 / a.group), all_lo_max = key_lo(a, seq, last / a.group),
              all_hi_min = key_hi(a, seq, r0 / a.group);
    const int w_lo = key_lo(a, seq, wfirst), w_lo_max = key_lo(a, seq, wlast),
              w_hi_min = key_hi(a, seq, wfirst), w_hi = key_hi(a, seq, wlast);
    const bool idle = r0 + 32 * mine > last;
    v8i qhi[S::DS], qlo[S::DS];
    const int qe = split_q<S::DS, 2, 16>(a.q + int64_t(seq.start + tok) * a.q_token +
                                         int64_t(kvh * a.group + head) * a.q_head + half * 32,
                                     64, a.q_mul, qhi, qlo);
    v16f o[S::DT];
#pragma unroll
    for (int i = 0; i < S::DT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (k0 < k1) {
      // a missing page anywhere in the run: every step looks for it
      bool hole = false;
      for (int p = (k0 >> a.page_bits) + int(threadIdx.x); p <= (k1 - 1) >> a.page_bits; p += 256)
        hole |= valid_page(a, table[p]) < 0;
      const bool holes = __syncthreads_or(hole);
      const int last_page = (k1 - 1) >> a.page_bits;
      auto page_at = [&](int key) {
        return table[min((key + 4 * kg) >> a.page_bits, last_page)];
      };
      auto is_masked = [&](int key) {
        return holes || key < all_lo_max || key + kManyKeys > all_hi_min;
      };
      ManyLoad<D> t;
      many_load<D>(a, kvh, k0, page_at(k0), t);
      int page = page_at(k0 + kManyKeys);
      many_store<D>(lds, t, k0, is_masked(k0), all_lo, keys.end, &nans);
      int cur = 0;
      for (int key = k0; key < k1; key += kManyKeys) {
        const bool more = key + kManyKeys < k1;
        if (more) {
          many_load<D>(a, kvh, key + kManyKeys, page, t);
          page = page_at(key + 2 * kManyKeys);
        }
        __syncthreads();  // this step's buffer is written, the other one read
        const uint8_t* buf = lds + cur * S::BUF;
        if (!idle && key < w_hi && key + kManyKeys > w_lo) {
          float p[KT][16];
          float top = -INFINITY;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const int krow = 32 * (kfirst + kt) + col;
            const int ks = buf[S::KB + S::VB + krow];
            v16f s = {};
#pragma unroll
            for (int d = 0; d < S::DS; ++d) {
              const uint4 x = *reinterpret_cast<const uint4*>(buf + k_at<D>(krow, 4 * d + 2 * half));
              const uint4 y =
                  *reinterpret_cast<const uint4*>(buf + k_at<D>(krow, 4 * d + 2 * half + 1));
              v8i k;
              k[0] = int(x.x); k[1] = int(x.y); k[2] = int(x.z); k[3] = int(x.w);
              k[4] = int(y.x); k[5] = int(y.y); k[6] = int(y.z); k[7] = int(y.w);
              s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, qhi[d], s, 0, 0, 0, ks, 0, qe);
              s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, qlo[d], s, 0, 0, 0, ks, 0, qe);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) p[kt][j] = s[j];
          }
          if (holes || key < w_lo_max || key + kManyKeys > w_hi_min) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const bool gone =
                    holes && *reinterpret_cast<const uint32_t*>(
                                 buf + S::KB + S::VB + 32 * (kfirst + kt) + 8 * g + 4 * half) == 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int kk = key + 32 * (kfirst + kt) + 8 * g + 4 * half + r;
                  if (gone || kk < lo || kk >= hi) p[kt][4 * g + r] = -INFINITY;
                }
              }
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, p[kt][j]);
          top = fmaxf(top, other_half(top));
          top = fmaxf(top, m);
          if (__ballot(top > m)) {
            const float f = top == m ? 1.0f : exp2_fast((m - top) * a.c);
            m = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < S::DT; ++i) o[i] *= f;
          }
          const float off = top == -INFINITY ? 0.0f : top * a.c;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              p[kt][j] = exp2_fast(__builtin_fmaf(p[kt][j], a.c, -off));
              l += p[kt][j];
            }
#pragma unroll
          for (int s = 0; s < 2 * KT; ++s) {
            const float* x = p[s >> 1] + 8 * (s & 1);
            const v8bf pf = as_bf(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                  pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
#pragma unroll
            for (int i = 0; i < S::DT; ++i) {
              const uint4 w = *reinterpret_cast<const uint4*>(
                  buf + S::KB + v_at(32 * i + col, 2 * (2 * kfirst + s) + half));
              o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf(w.x, w.y, w.z, w.w), pf, o[i],
                                                             0, 0, 0);
            }
          }
        }
        cur ^= 1;
        if (more)
          many_store<D>(lds + cur * S::BUF, t, key + kManyKeys, is_masked(key + kManyKeys), all_lo,
                        keys.end, &nans);
      }
      __syncthreads();  // (the next tile writes the buffers again)
      if constexpr (KS == 2) join_halves<S::DT, 2, 2 * S::BUF>(a, lds, wave, lane, o, m, l);
      mark_nan_rows<D>(a, table, kvh, nans, lo, hi, half, o);
    }
    l += other_half(l);
    if (wave < 4 / KS && r0 + 32 * mine + col <= last) {
      const int64_t at = int64_t(seq.start + tok) * a.heads + kvh * a.group + head;
      if (keys.live <= 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < S::DT; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(a.out + at * D + 32 * i + 8 * g + 4 * half) =
                make_uint2(pack_bf16(o[i][4 * g] * inv, o[i][4 * g + 1] * inv),
                           pack_bf16(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv));
      } else {
        const int64_t pa = int64_t(split) * a.tokens * a.heads + at;
#pragma unroll
        for (int i = 0; i < S::DT; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(a.part + pa * D + 32 * i + 8 * g + 4 * half) =
                make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        if (half == 0) {
          a.part_ml[2 * pa] = m;
          a.part_ml[2 * pa + 1] = l;
        }
      }
    }
  }
}

// ---- many rows, eight waves --------------------------------------------------
//
// As above (that chunk: 493-500 us, 1031-1046 TFLOP/s counting 4 flops a visible
// key, head and column, where a bf16 product of the library reaches 1245; heads
// of 64 319-321 us) with 256 rows a workgroup, so that each key is fetched, converted
// and written to LDS for twice the rows, and 128 keys between two barriers, so
// that the two waves of a SIMD drift apart and one's products run beside the
// other's softmax.  The codes of K need no work: each wave copies the 8 or 16
// rows it stages straight into LDS.  Keys staged by a wave lie in one page, so
// their addresses are the wave's own.
//
// KS == 2: 128 rows a workgroup; of the 128 keys each wave takes 64, four waves
// the even steps and four the odd ones, and the two sums of a row are joined
// through LDS at the end.  A wave alone on its SIMD takes 1.05 us a step (heads of
// 64), products and softmax in turn: a prompt of few tiles is as slow as its
// longest chain of steps, which this halves.
constexpr int kWideRows = 256;

template <int D>
struct WideShape {
  static constexpr int DS = D / 64, DT = D / 32;
  static constexpr int DG = D / 4;                      // threads across a row of codes
  static constexpr int KW = 256 / DG;                   // keys a wave stages of a 64-key step
  static constexpr int TU = D == 128 ? 2 : 1;           // steps that a thread stages
  static constexpr int KB = kManyKeys * D;              // bytes of K
  static constexpr int VB = kManyKeys * D * 2;          // and of V
  static constexpr int BUF = 2 * (KB + VB + kManyKeys); // two steps with their scales
};

// byte offset of chunk c (8 keys) of column d of V
TCFP_DEV int vp_at(int d, int c) { return d * 128 + ((c ^ ((d ^ ((d >> 3) & 3)) & 7)) << 4); }

// 16 bytes from base + off of each lane into LDS at lds + 16 * lane (base and
// lds the wave's); done when vmcnt has counted it.  (A copy into LDS needs one
// wait state behind the instruction that writes m0; the compiler, which sees to
// that for instructions of its own, does not look into the assembly.)
TCFP_DEV void copy_to_lds(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "{m0}"(lds)
               : "memory");
}

struct WideLoad {
  uint32_t v[4], ke, ve;
  int page;
};

template <int D, int KS>
__global__ __launch_bounds__(512, 2) void attend_wide_kernel(Attend a) {
  using S = WideShape<D>;
  constexpr int RT = kWideRows / KS;
  __shared__ uint4 lds4[2 * S::BUF / 16];
  __shared__ NanKeys nans;
  if (threadIdx.x == 0) nans = {INT32_MAX, 0};  // (a barrier follows before any step)
  uint8_t* const lds = reinterpret_cast<uint8_t*>(lds4);
  const uint32_t lds_at =
      uint32_t(uintptr_t((__attribute__((address_space(3))) uint8_t*)(lds4)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
            col = lane & 31, half = lane >> 5;
  int tile, split, kvh, b;
  if (!place(a, tile, split, kvh, b)) return;
  const Seq seq = sequence(a, b);
  if (split == 0 && tile == 0)
    zero_rest(a, b == 0 ? seq.start : 0,
              b == a.batch - 1 ? seq.start + seq.new_tokens : a.tokens, kvh * a.group, a.group, D);
  const int mine = wave % (8 / KS);  // the wave's 32 rows of the tile
  const int32_t* table = a.table + int64_t(b) * a.table_stride;
  // The wave stages keys 16 k16 + ... of a step: of K the rows kwave ... of
  // those 16, 16 bytes a lane (the chunk that belongs at the lane's place), of
  // V the thread's four keys 4 kg ..., one word of their rows each.  (The two or
  // four groups of four keys of a wave are dealt so that each half of it writes
  // both halves of the 16-byte chunks of V.)
  const int k16 = D == 128 ? wave >> 1 : wave & 3, kwave = D == 128 ? 8 * (wave & 1) : 0;
  const int krow_l = lane / (D / 16), kch = lane % (D / 16);
  const uint32_t koff =
      uint32_t(krow_l * D + ((kch ^ (D == 64 ? (krow_l >> 1) & 3 : krow_l & 7)) << 4));
  const int x4 = lane >> 4;
  const int kg = 4 * k16 + (D == 128 ? (wave & 1) + 2 * (x4 & 1) : ((x4 & 1) << 1) + (x4 >> 1));
  const int dg = (lane & 15) + (D == 128 ? (x4 >> 1) * 16 : 0);
  const int voff = (kg & 3) * 4 * D + dg * 4;
  const int vchunk = (kg >> 2) * 2 + (kg & 1), sub = ((kg >> 1) & 1) * 8;
  for (int r0 = tile * RT; r0 < seq.rows; r0 += a.tiles * RT) {
    const Keys keys = keys_of(a, seq, r0, RT);
    if (split >= max(keys.live, 1)) continue;
    const int k0 = keys.begin + split * a.chunk;
    const int k1 = split == a.splits - 1 ? keys.end : min(keys.end, k0 + a.chunk);
    const int last = min(r0 + RT, seq.rows) - 1;
    const int row = min(r0 + 32 * mine + col, last), tok = row / a.group,
              head = row - tok * a.group;
    const int lo = key_lo(a, seq, tok), hi = key_hi(a, seq, tok);
    const int wfirst = min(r0 + 32 * mine, last) / a.group,
              wlast = min(r0 + 32 * mine + 31, last) / a.group;
    const int all_lo = key_lo(a, seq, r0 / a.group), all_lo_max = key_lo(a, seq, last / a.group),
              all_hi_min = key_hi(a, seq, r0 / a.group);
    const int w_lo = key_lo(a, seq, wfirst), w_lo_max = key_lo(a, seq, wlast),
              w_hi_min = key_hi(a, seq, wfirst), w_hi = key_hi(a, seq, wlast);
    const bool idle = r0 + 32 * mine > last;
    v8i qhi[S::DS], qlo[S::DS];
    const int qe = split_q<S::DS, 2, 16>(a.q + int64_t(seq.start + tok) * a.q_token +
                                         int64_t(kvh * a.group + head) * a.q_head + half * 32,
                                     64, a.q_mul, qhi, qlo);
    v16f o[S::DT];
#pragma unroll
    for (int i = 0; i < S::DT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (k0 < k1) {
      const int last_page = (k1 - 1) >> a.page_bits;
      bool hole = false;
      for (int p = (k0 >> a.page_bits) + int(threadIdx.x); p <= last_page; p += 512)
        hole |= valid_page(a, table[p]) < 0;
      const bool holes = __syncthreads_or(hole);
      auto is_masked = [&](int key) {
        return holes || key < all_lo_max || key + kManyKeys > all_hi_min;
      };
      // the page of the wave's keys of a step (as read; made scalar at its use)
      auto page_of = [&](int key) { return table[min((key + 16 * k16) >> a.page_bits, last_page)]; };
      auto step_of = [&](int i) { return D == 128 ? i : wave >> 2; };
      WideLoad t[S::TU];
      int page[S::TU];
      // keys of the steps at key0 on their way: K to LDS, V to registers
      auto fetch = [&](int key0, uint32_t buf) {
#pragma unroll
        for (int i = 0; i < S::TU; ++i) {
          const int u = step_of(i), key = key0 + u * kManyKeys;
          const int pg = __builtin_amdgcn_readfirstlane(valid_page(a, page[i]));
          t[i].page = pg;
          const int64_t at = ((int64_t(max(pg, 0)) * a.kv_heads + kvh) << a.page_bits) +
                             ((key + 16 * k16) & ((1 << a.page_bits) - 1));
          copy_to_lds(a.k_codes + (at + kwave) * D, koff,
                      buf + uint32_t(u * S::KB + (16 * k16 + kwave) * D));
          const uint8_t* v = a.v_codes + at * D + voff;
#pragma unroll
          for (int j = 0; j < 4; ++j) t[i].v[j] = *reinterpret_cast<const uint32_t*>(v + j * D);
          t[i].ke = *reinterpret_cast<const uint32_t*>(a.k_exps + at + (kg & 3) * 4);
          t[i].ve = *reinterpret_cast<const uint32_t*>(a.v_exps + at + (kg & 3) * 4);
          page[i] = page_of(key + 2 * kManyKeys);
        }
      };
      // what fetch() brought, complete in the buffer but for a barrier
      auto settle = [&](int key0, uint8_t* buf) {
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
#pragma unroll
        for (int i = 0; i < S::TU; ++i) {
          const int u = step_of(i), key = key0 + u * kManyKeys;
          uint32_t scales = ((t[i].ke & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) ^ (t[i].ke & 0x80808080u);
          if (is_masked(key)) {
            bool nan = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int kk = key + 4 * kg + j;
              const bool dead = kk < all_lo || kk >= keys.end || t[i].page < 0;
              if (dead) t[i].v[j] = 0;
              nan |= nan_bytes(t[i].v[j]) != 0;
              t[i].v[j] = without_nan(t[i].v[j]);
              if (dead) t[i].ve &= ~(0xFFu << (8 * j));
            }
            if (nan) note_nan(&nans, key, kManyKeys);
            if (t[i].page < 0) scales = 0;
          }
          float sc[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[j] = exp_scale(t[i].ve, j);
          uint8_t* vb = buf + 2 * S::KB + u * S::VB + sub;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x[j] = h ? deq2<true>(t[i].v[j], sc[j]) : deq2<false>(t[i].v[j], sc[j]);
            *reinterpret_cast<uint2*>(vb + vp_at(dg * 4 + 2 * h, vchunk)) =
                make_uint2(lows(x[0], x[1]), lows(x[2], x[3]));
            *reinterpret_cast<uint2*>(vb + vp_at(dg * 4 + 2 * h + 1, vchunk)) =
                make_uint2(highs(x[0], x[1]), highs(x[2], x[3]));
          }
          if (dg == 0)
            *reinterpret_cast<uint32_t*>(buf + 2 * (S::KB + S::VB) + u * kManyKeys + 4 * kg) = scales;
        }
      };
#pragma unroll
      for (int i = 0; i < S::TU; ++i) page[i] = page_of(k0 + step_of(i) * kManyKeys);
      fetch(k0, lds_at);
      settle(k0, lds);
      int cur = 0;
      for (int key0 = k0; key0 < k1; key0 += 2 * kManyKeys) {
        const bool more = key0 + 2 * kManyKeys < k1;
        __syncthreads();  // this buffer is written, the other one read
        if (more) fetch(key0 + 2 * kManyKeys, lds_at + uint32_t((cur ^ 1) * S::BUF));
#pragma unroll 1
        for (int u = wave / (8 / KS); u < 2; u += KS) {
          const int key = key0 + u * kManyKeys;
          if (idle || key >= w_hi || key + kManyKeys <= w_lo || key >= k1) continue;
          const uint8_t* buf = lds + cur * S::BUF + u * S::KB;
          const uint8_t* vb = lds + cur * S::BUF + 2 * S::KB + u * S::VB;
          const uint8_t* sb = lds + cur * S::BUF + 2 * (S::KB + S::VB) + u * kManyKeys;
          // (a wave at its products goes first: 498 -> 493 us)
          __builtin_amdgcn_s_setprio(1);
          v16f s[2];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            const int krow = 32 * kt + col;
            const int ks = sb[krow];
            s[kt] = v16f{};
#pragma unroll
            for (int d = 0; d < S::DS; ++d) {
              const uint4 x = *reinterpret_cast<const uint4*>(buf + k_at<D>(krow, 4 * d + 2 * half));
              const uint4 y =
                  *reinterpret_cast<const uint4*>(buf + k_at<D>(krow, 4 * d + 2 * half + 1));
              v8i k;
              k[0] = int(x.x); k[1] = int(x.y); k[2] = int(x.z); k[3] = int(x.w);
              k[4] = int(y.x); k[5] = int(y.y); k[6] = int(y.z); k[7] = int(y.w);
              s[kt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, qhi[d], s[kt], 0, 0, 0, ks,
                                                                      0, qe);
              s[kt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, qlo[d], s[kt], 0, 0, 0, ks,
                                                                      0, qe);
            }
          }
          __builtin_amdgcn_s_setprio(0);
          if (holes || key < w_lo_max || key + kManyKeys > w_hi_min) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const bool gone = holes && *reinterpret_cast<const uint32_t*>(
                                               sb + 32 * kt + 8 * g + 4 * half) == 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int kk = key + 32 * kt + 8 * g + 4 * half + r;
                  if (gone || kk < lo || kk >= hi) s[kt][4 * g + r] = -INFINITY;
                }
              }
          }
          float top = s[0][0];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int x = 0; x < 16; ++x) top = fmaxf(top, s[kt][x]);
          top = fmaxf(top, other_half(top));
          top = fmaxf(top, m);
          if (__ballot(top > m)) {
            const float f = top == m ? 1.0f : exp2_fast((m - top) * a.c);
            m = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < S::DT; ++i) o[i] *= f;
          }
          const float off = top == -INFINITY ? 0.0f : top * a.c;
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              s[kt][x] = exp2_fast(__builtin_fmaf(s[kt][x], a.c, -off));
              l += s[kt][x];
            }

#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const v16f& e = s[x >> 1];
            const int z = 8 * (x & 1);
            const v8bf p = as_bf(pack_bf16(e[z], e[z + 1]), pack_bf16(e[z + 2], e[z + 3]),
                         pack_bf16(e[z + 4], e[z + 5]), pack_bf16(e[z + 6], e[z + 7]));
#pragma unroll
            for (int i = 0; i < S::DT; ++i) {
              const uint4 w = *reinterpret_cast<const uint4*>(vb + vp_at(col, 2 * x + half) + 4096 * i);
              o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf(w.x, w.y, w.z, w.w), p, o[i],
                                                             0, 0, 0);
            }
          }
        }
        cur ^= 1;
        if (more) settle(key0 + 2 * kManyKeys, lds + cur * S::BUF);
      }
      __syncthreads();  // (the next tile writes the buffers again)
      if constexpr (KS == 2) join_halves<S::DT, 4, 2 * S::BUF>(a, lds, wave, lane, o, m, l);
      mark_nan_rows<D>(a, table, kvh, nans, lo, hi, half, o);
    }
    l += other_half(l);
    if (wave < 8 / KS && r0 + 32 * mine + col <= last) {
      const int64_t at = int64_t(seq.start + tok) * a.heads + kvh * a.group + head;
      if (keys.live <= 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < S::DT; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(a.out + at * D + 32 * i + 8 * g + 4 * half) =
                make_uint2(pack_bf16(o[i][4 * g] * inv, o[i][4 * g + 1] * inv),
                           pack_bf16(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv));
      } else {
        const int64_t pa = int64_t(split) * a.tokens * a.heads + at;
#pragma unroll
        for (int i = 0; i < S::DT; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(a.part + pa * D + 32 * i + 8 * g + 4 * half) =
                make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        if (half == 0) {
          a.part_ml[2 * pa] = m;
          a.part_ml[2 * pa + 1] = l;
        }
      }
    }
  }
}

// W waves a row: the parts of its item, if it has several.  Each wave takes every
// W-th part with a running maximum, then the waves are joined in order.  Four waves
// where there are few rows, each with many parts; one where the rows fill the
// card, which then has a quarter of the waves to start, each of which looks for
// its item among all sequences (64 x 32 rows 8.6 -> 5.5 us, with the attention
// itself 134.8 -> 131.2; 200 x 16 rows 47.3 -> 42.4 in all; 4 x 16 rows 15.0 -> 15.7).
template <int D, int W>
__global__ __launch_bounds__(256) void attend_few_join_kernel(Attend a, int tile_rows) {
  constexpr int C = D / 64, R = 4 / W;  // columns of a lane, rows of a workgroup
  __shared__ FindLds fl;
  __shared__ float ml[4][2];
  __shared__ float xo[4][D];
  const int lane = threadIdx.x & 63, wave = scalar(int(threadIdx.x >> 6));
  const unsigned groups = unsigned(a.heads + R - 1) / R, t_ = blockIdx.x / groups;
  const int t = int(t_), h = int(blockIdx.x - t_ * groups) * R + wave / W, first_wave = wave % W;
  Found at;
  const bool any = find(
      a, tile_rows, fl,
      [&](const Seq& s, int64_t, int64_t, int64_t) {
        return t >= s.start && t < s.start + s.new_tokens;
      },
      at);
  if (!any || h >= a.heads) return;  // (h: of all waves or, alone, of this one)
  const int64_t share = share_of(a, at.total);
  const int r = (t - at.seq.start) * a.group + h % a.group, units = units_of(a, at.seq);
  const int64_t first =
      at.before + int64_t(r / tile_rows * a.kv_heads + h / a.group) * units;  // the item's first unit
  // (bounded: sequences whose rows overlap, which no batch has, would be found as a
  // mixture of several, and their parts nowhere)
  const int64_t most = a.workers - 1;
  const int w0 = int(min(divide(first, share), most)),
            w1 = int(min(divide(first + units - 1, share), most));
  if (w0 == w1) return;
  float m = -INFINITY, l = 0.0f, o[C] = {};
  constexpr int N = 4;  // parts of a wave in flight
  for (int w = w0 + first_wave; w <= w1; w += W * N) {
    float pm[N], pl[N], po[N][C];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = min(w + W * i, w1);
      const int64_t p = (2 * int64_t(x) + (x == w0 ? 1 : 0)) * tile_rows + r % tile_rows;
      pm[i] = a.part_ml[2 * p];
      pl[i] = a.part_ml[2 * p + 1];
#pragma unroll
      for (int c = 0; c < C; ++c) po[i][c] = a.part[p * D + lane * C + c];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (w + W * i > w1) continue;
      const float top = fmaxf(m, pm[i]);
      const float f = m == top ? 1.0f : exp2_fast((m - top) * a.c);
      const float g = pm[i] == top ? 1.0f : exp2_fast((pm[i] - top) * a.c);
      m = top;
      l = l * f + pl[i] * g;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = o[c] * f + po[i][c] * g;
    }
  }
  uint16_t* const out = a.out + (int64_t(t) * a.heads + h) * D;
  if constexpr (W == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < C; ++c) out[lane * C + c] = f32_to_bf16_rne(o[c] * inv);
    return;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) xo[wave][lane * C + c] = o[c];
  if (lane == 0) {
    ml[wave][0] = m;
    ml[wave][1] = l;
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][0]);
  float sum = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = ml[w][0] == top ? 1.0f : exp2_fast((ml[w][0] - top) * a.c);
    sum += ml[w][1] * f[w];
  }
  if (threadIdx.x < D) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v += xo[w][threadIdx.x] * f[w];
    out[threadIdx.x] = f32_to_bf16_rne(sum == 0.0f ? 0.0f : v / sum);
  }
}

// A wave a row whose keys were split: the splits' sums, brought to the largest
// maximum and added in order.
template <int D>
__global__ __launch_bounds__(256) void attend_join_kernel(Attend a, int tile_rows) {
  constexpr int C = D / 64;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t rows = int64_t(a.tokens) * a.heads;
  if (row >= rows) return;
  const int t = int(row / a.heads), h = int(row - int64_t(t) * a.heads);
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const Seq seq = sequence(a, lo);
  if (t < seq.start || t >= seq.start + seq.new_tokens) return;
  const int r = (t - seq.start) * a.group + h % a.group;
  const Keys keys = keys_of(a, seq, r / tile_rows * tile_rows, tile_rows);
  if (keys.live <= 1) return;
  float m = -INFINITY, l = 0.0f;
  if (lane < keys.live) {
    m = a.part_ml[2 * (lane * rows + row)];
    l = a.part_ml[2 * (lane * rows + row) + 1];
  }
  const float top = wave_max(m);
  const float f = m == top ? 1.0f : exp2_fast((m - top) * a.c);
  float sum = l * f;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
  float o[C] = {};
  for (int s = 0; s < keys.live; ++s) {
    const float fs = __shfl(f, s, 64);
    const float* p = a.part + (s * rows + row) * D + lane * C;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] += fs * p[c];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < C; ++c) a.out[row * D + lane * C + c] = f32_to_bf16_rne(o[c] * inv);
}

// How the batch is laid over the card, from the bounds of its lengths.
struct Launch {
  int few_tiles;  // 16-row tiles a workgroup of the few-rows kernel takes; 0: many rows
  bool wide;      // 256 rows a workgroup
  bool paired;    // 128 rows of eight waves, 64 of four for heads of 256
  int tile_rows, tiles, splits, chunk;
  int workers;    // few rows: workgroups
  bool whole;     // few rows: one workgroup an item
};
Launch plan(int64_t tokens, int heads, int kv_heads, int dim, int64_t batch,
            int64_t max_query_len, int64_t max_seq_len, int64_t window) {
  Launch p{};
  // (a window past every position is none, a bound past every length no bound;
  // sums of larger ones would overflow)
  window = std::min(window, kMostKeys);
  max_query_len = std::min(max_query_len, kMostKeys);
  const int64_t group = heads / kv_heads;
  const int64_t most = std::max<int64_t>(std::min(max_query_len, tokens), 1) * group;
  int64_t keys = std::clamp<int64_t>(max_seq_len, 1, kMostKeys);
  if (window > 0) keys = std::min(keys, window + max_query_len + 64);
  p.few_tiles = most <= 16 ? 1 : most <= 32 ? 2 : 0;
  if (p.few_tiles) {
    p.tile_rows = 16 * p.few_tiles;
    p.tiles = 1;
    // two workgroups a CU, one for heads of 256, which need twice the registers
    // (64 sequences of up to 8192 tokens, 16 / 8 heads of 256: 449 us with spills
    // at two, 248 us at one), fewer where there is less to do
    const int64_t items = batch * kv_heads;
    p.whole = keys <= 2 * kUnit;
    const int64_t units = p.whole ? items : items * ((keys + kUnit - 1) / kUnit + 1);
    p.workers = int(std::min<int64_t>(units, dim == 256 ? 256 : 512));
    p.splits = p.whole ? 1 : 2;
    return p;
  }
  // workgroups without splitting: at most one tile a sequence is part full
  auto workgroups = [&](int64_t rows) {
    const int64_t tiles = (most + rows - 1) / rows * batch;
    return std::max<int64_t>(std::min(tiles, tokens * group / rows + batch) * kv_heads, 1);
  };
  // 256 rows a workgroup where all tiles see about as many keys (as much cached
  // before the new tokens as there are of these) or there are many rounds of
  // them; else 128, two workgroups a CU, which even out the tiles of a causal
  // prompt (one of 2048 tokens, 32 / 8 heads of 128: 66.6 us against 76.2; four
  // of up to 500: 25.7 against 29.6; 2048 over 14336: 553 against 493).
  p.wide = dim <= 128 && most > kWideRows &&
           (keys >= 2 * max_query_len || workgroups(kWideRows) >= 512);
  // Eight waves on 128 rows, which halves the chain of a tile's steps, where
  // there are tiles for a good part of the CUs and for no CU two, and the longest
  // is not short (one prompt of 1000 tokens, 16 heads of 64: 24.7 -> 19.7 us; of
  // 2048, 8 / 2 heads of 128: 47.1 -> 38.7; six of up to 1000, 16 heads of 64, 480
  // tiles: 32.8 against 40.0; 600 over 300, 4 heads of 128, 20 tiles: 21.3 against
  // 23.1, as fewer runs fill the card; 256, 32 / 8 heads of 128: 14.8 against 15.7).
  const int64_t tiles = workgroups(kManyRows);
  p.paired = !p.wide && keys >= 512 && tiles > 64 && tiles <= 256;
  p.tile_rows = p.wide ? kWideRows : kManyRows;
  if (dim == 256) {
    // (64 rows of four waves, each with half of a step's keys; 100 tokens, 8 heads:
    // 20.7 -> 16.2 us, 777 over 100, 6 / 2 heads: 64.1 -> 53.6; a long context is
    // better split: 426 over 1218, 3 heads on one: 37.5 against 50.7)
    p.paired = keys <= 1536 && workgroups(kManyRows / 2) <= 256;
    if (p.paired) p.tile_rows = kManyRows / 2;
  }
  p.tiles = int((most + p.tile_rows - 1) / p.tile_rows);
  // Splits of the keys, as many as there is room for at most, by what they are
  // about to take: a workgroup's pass over its keys, 0.21 ns a key and column (64
  // keys of 64, 128 and 256 columns: 1.1, 1.75 and 3.6 us); writing and joining
  // the parts, 3 TB/s; another launch, 5 us.  (A causal prompt of 1000 tokens, 32
  // / 8 heads of 128: 36.3 us whole, 47.8 in two; 64 tokens over 4000: 105 whole,
  // 28.7 in 12 runs, 34.8 in 32; 512 over 4096, 8 / 2 heads of 256: 61.7 in 8 runs,
  // which fill the card once, 79.0 in 16.)
  const int64_t room = (p.wide || p.paired || dim == 256 ? 256 : 512) / workgroups(p.tile_rows);
  const double pass = 0.21 * double(keys) * dim, part = double(tokens) * heads * dim * 8 / 3000;
  int64_t splits = 1;
  double least = pass;
  for (int64_t n = 2; n <= std::min<int64_t>(room, kMaxSplits); ++n) {
    const double t = pass / double(n) + part * double(n) + 5000;
    if (t < least) least = t, splits = n;
  }
  p.chunk = int(((keys + splits - 1) / splits + 127) / 128 * 128);
  p.splits = int(std::clamp<int64_t>((keys + p.chunk - 1) / p.chunk, 1, kMaxSplits));
  return p;
}

// Rows that parts are kept of.
int64_t part_rows(const Launch& p, int64_t tokens, int heads) {
  if (p.splits <= 1) return 0;
  return p.few_tiles ? 2 * int64_t(p.workers) * p.tile_rows : p.splits * tokens * heads;
}
size_t workspace_of(const Launch& p, int64_t tokens, int heads, int dim) {
  return size_t(part_rows(p, tokens, heads)) * size_t(dim + 2) * sizeof(float);
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
                                            int64_t max_seq_len, int64_t window) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  return workspace_of(
      plan(tokens, heads, kv_heads, dim, batch, max_query_len, max_seq_len, window), tokens, heads,
      dim);
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
      window < 0 || tokens * (heads / kv_heads) > INT32_MAX / 2)
    return TCFP_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_codes) || !aligned16(v_codes) ||
      q_token_stride % 8 || q_head_stride % 8 || (reinterpret_cast<uintptr_t>(k_exps) & 3u) ||
      (reinterpret_cast<uintptr_t>(v_exps) & 3u))
    return TCFP_ERR_ALIGN;
  if (tokens == 0) return TCFP_OK;
  if (batch == 0) return TCFP_ERR_SHAPE;
  const Launch p =
      plan(tokens, heads, kv_heads, dim, batch, max_query_len, max_seq_len, window);
  const size_t need = workspace_of(p, tokens, heads, dim);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return TCFP_ERR_WORKSPACE;
  Attend a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_exps = k_exps;
  a.v_exps = v_exps;
  a.num_pages = int(num_pages);
  a.page_bits = log2i(page_size);
  a.kv_heads = kv_heads;
  a.table = page_table;
  a.table_stride = table_stride;
  // (a pool without pages holds no key)
  a.table_keys = num_pages == 0 ? 0 : int(std::min<int64_t>(table_width * page_size, kMostKeys));
  a.seq_lens = seq_lens;
  a.starts = query_start;
  a.batch = int(batch);
  a.tokens = int(tokens);
  a.heads = heads;
  a.group = heads / kv_heads;
  a.c = scale == 0.0f ? 1.0f : std::abs(scale) * 1.44269504088896340736f;
  a.q_mul = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
  a.causal = causal != 0;
  a.window = int(std::min<int64_t>(window, kMostKeys));
  a.tiles = p.tiles;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + part_rows(p, tokens, heads) * dim;
  a.workers = p.workers;
  a.whole = p.whole;
  const auto st = static_cast<hipStream_t>(stream);
#define TCFP_BY_DIM(CALL)         \
  do {                            \
    if (dim == 64) CALL(64);      \
    else if (dim == 128) CALL(128); \
    else CALL(256);               \
  } while (0)
  if (p.few_tiles) {
#define TCFP_FEW(D)                                                       \
  do {                                                                    \
    if (p.few_tiles == 1) attend_few_kernel<D, 1><<<p.workers, 256, 0, st>>>(a); \
    else attend_few_kernel<D, 2><<<p.workers, 256, 0, st>>>(a);                \
  } while (0)
    TCFP_BY_DIM(TCFP_FEW);
#undef TCFP_FEW
  } else {
    const int64_t sets = int64_t(p.splits) * kv_heads * batch;
    const int64_t wgs = p.tiles * (sets >= 8 ? (sets + 7) / 8 * 8 : sets);
    a.sets = int(std::min<int64_t>(sets, INT32_MAX));
    // (half of an XCD's 4 MiB)
    a.tiles_first = (sets + 7) / 8 * std::min<int64_t>(p.chunk, max_seq_len) * dim * 2 <= 2 << 20;
    if (wgs > INT32_MAX || !grid_x_fits(wgs, 512)) return TCFP_ERR_SHAPE;
#define TCFP_MANY(D) attend_many_kernel<D, 1><<<unsigned(wgs), 256, 0, st>>>(a)
    if (p.wide && dim == 64) attend_wide_kernel<64, 1><<<unsigned(wgs), 512, 0, st>>>(a);
    else if (p.wide) attend_wide_kernel<128, 1><<<unsigned(wgs), 512, 0, st>>>(a);
    else if (p.paired && dim == 64) attend_wide_kernel<64, 2><<<unsigned(wgs), 512, 0, st>>>(a);
    else if (p.paired && dim == 128) attend_wide_kernel<128, 2><<<unsigned(wgs), 512, 0, st>>>(a);
    else if (p.paired) attend_many_kernel<256, 2><<<unsigned(wgs), 256, 0, st>>>(a);
    else TCFP_BY_DIM(TCFP_MANY);
#undef TCFP_MANY
  }
  if (p.splits > 1 && p.few_tiles) {
    const int64_t rows = tokens * heads, quarter = tokens * ((heads + 3) / 4);
    if (!grid_x_fits(rows, 256)) return TCFP_ERR_SHAPE;
#define TCFP_JOIN(D)                                                            \
  do {                                                                          \
    if (rows > 1024)                                                            \
      attend_few_join_kernel<D, 1>                                              \
          <<<unsigned(quarter), 256, 0, st>>>(a, p.tile_rows);                  \
    else                                                                        \
      attend_few_join_kernel<D, 4><<<unsigned(rows), 256, 0, st>>>(a, p.tile_rows); \
  } while (0)
    TCFP_BY_DIM(TCFP_JOIN);
#undef TCFP_JOIN
  } else if (p.splits > 1) {
    const int64_t blocks = (tokens * heads + 3) / 4;
    if (!grid_x_fits(blocks, 256)) return TCFP_ERR_SHAPE;
#define TCFP_JOIN(D) attend_join_kernel<D><<<unsigned(blocks), 256, 0, st>>>(a, p.tile_rows)
    TCFP_BY_DIM(TCFP_JOIN);
#undef TCFP_JOIN
  }
#undef TCFP_BY_DIM
  return launch_status();
}

}  // extern "C"
