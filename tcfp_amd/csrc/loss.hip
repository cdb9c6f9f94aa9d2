// Softmax cross entropy of a linear head over a large vocabulary, and its
// gradients (gfx950).
//
//   z = h W^T,  lse = log sum exp z,  loss = lse - z[target]
//   g = (softmax(z) - onehot(target)) * grad / unit,  dh = unit g W,  dW = unit g^T h
//
// (unit: the gradient of a sum, that of a mean over the tokens that count, or the
// largest of all tokens'.  With it in g, every g of a target would be the same number
// near -unit, whose rounding to bf16 all tokens' gradients would share: 3.6e-3 off
// where the results' own rounding is 1.7e-3.)
// h [tokens, dim] and W [vocab, dim] are bf16.  Forward: one product whose epilogue
// reduces every 256 (128) classes of a token to their maximum and sum of
// exponentials, which a small launch joins; z is not stored.
//
// Exponentials are of differences from the maximum, formed before they are scaled to
// powers of two, and the loss is (maximum - z[target]) + log(sum): right to 2^-23 or so
// whatever the logits' size, and never below 0.  As lse - z[target], with lse rounded, it
// would be off by 2^-24 of lse: of 30, by 1.8e-6, as much as a confident token's whole
// loss.  The gradient of the target's logit, p - 1, is formed from the loss as exp(-loss)
// - 1.  Other classes' p = exp(z - lse) are off in proportion to themselves, by 2^-24 of
// lse for its rounding and as much for that of its multiple, about what z's own rounding
// to fp32 is: of 2000, 2e-4.
//
// Gradients, where they are wanted of the losses' sum or mean and tokens x classes
// take at most 1 GiB of workspace in 16 bits: with the forward, three products in
// all.  The first one's epilogue leaves 2^15 exp(z - maximum of its tile) in fp16 (11
// bits, as it is rounded once more; down to 2^-29 of the maximum, fewer to 2^-39: rare
// classes keep their gradients), a pass turns it into g in bf16 in place, and g is the
// operand of dh and dW.  Otherwise (more, or a gradient for every token's
// loss) the backward forms z again for a run of classes at a time, with g as the
// epilogue: dh is added up over the runs in fp32, of dW a run has its rows.  g is
// rounded to bf16 (2^-8 of each value at most, as the results themselves are); all sums
// are fp32.
#include <algorithm>
#include <cmath>
#include <utility>

#include "mfma_tiles.h"

using namespace tcfp;

namespace {

// ---- the products -----------------------------------------------------------
//
// C[n][m] = sum over k of B[n][k] A[m][k] with both operands read as they lie in
// memory: rows along k, or (TA, TB) rows of one k each, which LDS transposes on
// the way into the registers.  So W serves z = h W^T and dh = g W, and g serves
// dh = g W and dW = g^T h, without transposed copies.
//
// A workgroup owns T x T of C over a run of k (a split).  T = 256: eight waves, 2
// along m and 4 along n, 128 x 64 each; two stages of 64 k in LDS (128 KiB); one
// workgroup a CU, which takes tile after tile: the next one's first stages are on
// their way while a result is written, and its stores drain while the next one is
// multiplied (8192 x 32768 over 4096 with the exponentials, a workgroup a tile:
// 2066 us, so: 1886).  T = 128: four waves of 64 x 64; four stages (one workgroup
// a CU: what streams one operand from HBM, or has few tiles) or two (two workgroups,
// of which one multiplies while the other waits or stores).  cost() says which is
// taken.  A stage's copies are issued as soon as every wave has read its last operands
// of the stage whose place they take, in the middle of that stage's products.
constexpr int kStageK = 64;

TCFP_DEV uint32_t half2(float a, float b) {
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  const v2h v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, v);
}

template <int T, int ST>
struct Shape {
  static constexpr int WAVES = T == 256 ? 8 : 4, THREADS = 64 * WAVES;
  static constexpr int STAGES = ST;
  static constexpr int MB = T / 64, NB = 2;  // 32-row and 32-column blocks of a wave
  static constexpr int WAVES_M = 2;
  static constexpr int OPERAND = T * kStageK * 2, STAGE = 2 * OPERAND;
};

struct Product {
  const uint16_t *a, *b;
  int64_t lda, ldb;  // elements
  int m, n, k;
  int tiles_m, tiles_n;
  int splits, k_run; // of k, the latter a multiple of 64
  // results: bf16 or fp32 [n, m], rows ldo apart
  void* out;
  int64_t ldo;
  int64_t split_stride;
  int add;           // fp32: to what is there
  // the loss
  const int64_t* targets;
  int64_t ignore;
  int64_t first;     // class of m = 0
  int64_t classes;   // of the whole vocabulary
  float2* part;      // [tiles_m, n]: maximum, sum
  float* picked;     // [n]: z of the target
  int* done;         // cleared for the launch that joins the parts
  const float* lse;
  const float* losses;     // nullptr: the target's p - 1 from lse
  const float* grad;       // nullptr, or one a token, divided by *up
  const float *up, *over;  // unit is *up / *over, nullptr: 1 (bf16 results are times unit)
};
TCFP_DEV float unit_of(const float* up, const float* over) {
  const float u = up ? *up : 1.0f, o = over ? *over : 1.0f;
  return o == 0.0f ? 0.0f : u / o;  // (no tokens that count: no gradients)
}

// exp(-loss) - 1, to 2^-22 of itself: below 0.05 by its series, of which the next term is
// 5e-8.
TCFP_DEV float less_one(float loss) {
  const float x = -loss;
  return loss < 0.05f ? x * (1.0f + x * (0.5f + x * (1.0f / 6 + x * (1.0f / 24))))
                      : exp2_fast(x * kLog2e) - 1.0f;
}

// What the exponentials, 1 at most, are stored times.
constexpr float kExpsUp = 32768.0f;

// kStats: parts of the losses; kExps: those and the exponentials; kGrad: g.
enum Epilogue { kBf16, kFp32, kStats, kExps, kGrad };

// One operand's copies into LDS: 4 instructions a wave and stage.
// Rows along k: instruction q brings the rows 8 q ... of 128 bytes, whose eight
// chunks of 16 bytes are permuted by (row / 2) % 8; rows of one k: instruction q
// brings 1024 / (2 T) rows, whose chunks are permuted by 4 (row % 4), so that the
// reads meet every bank once.
template <int T, bool OF_K>
struct Copies {
  uint32_t off0, off1, step;  // of even and odd instructions
  int at0, at1;               // their chunks' first k (column)
  TCFP_DEV void init(int wave, int lane, int64_t ld) {
    constexpr int CH = OF_K ? T / 8 : 8, R = 64 / CH;  // chunks of a row, rows an instruction
    const int row = 4 * R * wave + lane / CH;
    int c0, c1;
    if constexpr (OF_K) {
      c0 = (lane % CH) ^ (4 * ((lane / CH) & 3));
      c1 = (lane % CH) ^ (4 * ((R + lane / CH) & 3));
    } else {
      c0 = (lane & 7) ^ ((lane >> 4) & 7);
      c1 = (lane & 7) ^ ((4 + (lane >> 4)) & 7);
    }
    off0 = uint32_t(row * ld * 2) + c0 * 16;
    off1 = uint32_t(row * ld * 2) + c1 * 16;
    step = uint32_t(R * ld * 2);
    at0 = c0 * 8;
    at1 = c1 * 8;
  }
  // The stage at k of rows (columns) [at, extent), k up to k1, into LDS at `to`; nothing
  // but zeros from k1 on.  (Whole chunks of 16 bytes: behind an odd number of classes g
  // has zeros.)
  TCFP_DEV void issue(const uint16_t* p, int64_t ld, int at, int extent, int k, int k1,
                      uint32_t to) const {
    const uint16_t* base;
    int64_t span;
    int left;  // of what a row holds
    if constexpr (OF_K) {
      base = p + int64_t(k) * ld + at;
      left = extent - at;
      span = (int64_t(min(k1 - k, kStageK)) - 1) * ld + ((left + 7) & ~7);
    } else {
      base = p + int64_t(at) * ld + k;
      left = k1 - k;
      span = (int64_t(min(extent - at, T)) - 1) * ld + ((left + 7) & ~7);
    }
    const v4i rsrc = make_rsrc(base, k < k1 ? uint32_t(span * 2) : 0u);
    const uint32_t o0 = at0 >= left ? kOutOfRange : off0, o1 = at1 >= left ? kOutOfRange : off1;
#pragma unroll
    for (int i = 0; i < 4; ++i) copy16(rsrc, ((i & 1) ? o1 : o0) + i * step, to + i * 1024);
  }
};

// What of C a workgroup computes.
struct Unit {
  int m0, n0, k0, k1, split, stages;
};
// Each XCD (workgroup b is on XCD b % 8) takes a run of the splits' tiles, in groups of
// four tile rows along n, so that its L2 holds both operands' panels.
template <int T>
TCFP_DEV Unit unit_at(const Product& g, int l) {
  Unit u;
  const int tiles = g.tiles_m * g.tiles_n, units = tiles * g.splits;
  l = (l & 7) * (units >> 3) + min(l & 7, units & 7) + (l >> 3);
  u.split = l / tiles;
  l -= u.split * tiles;
  const int per = 4 * g.tiles_m, first = l / per * 4, rows = min(g.tiles_n - first, 4);
  u.n0 = (first + l % per % rows) * T;
  u.m0 = l % per / rows * T;
  u.k0 = u.split * g.k_run;
  u.k1 = min(g.k, u.k0 + g.k_run);
  // (two at least, of which a second one may be zeros)
  u.stages = max((u.k1 - u.k0 + kStageK - 1) / kStageK, T == 256 ? 2 : 0);
  return u;
}

// Waits for the wave's LDS operations, then for the workgroup; copies and stores go on.
TCFP_DEV void sync_lds() { wait_and_sync<63>(); }

template <int T, int ST, bool TA, bool TB, int EPI>
__global__ __launch_bounds__(T == 256 ? 512 : 256, T == 128 && ST == 2 ? 2 : 1) void product_kernel(
    Product g) {
  using S = Shape<T, ST>;
  constexpr bool STATS = EPI == kStats || EPI == kExps, MANY = T == 256;
  // Of each wave 4 KiB beside the stages (or, where the workgroup has one tile, in their
  // place when they are done with): what the epilogue takes, and its result on its way
  // to rows.
  constexpr int PRIVATE = 4096;
  __shared__ __align__(16) uint8_t lds[S::STAGES * S::STAGE + (MANY ? S::WAVES * PRIVATE : 0)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int wm = wave % S::WAVES_M, wn = wave / S::WAVES_M;
  uint8_t* const spare = lds + (MANY ? S::STAGES * S::STAGE : 0);
  uint8_t* const own = spare + wave * PRIVATE;
  if (STATS && blockIdx.x == 0 && threadIdx.x == 0) *g.done = 0;

  // (kept in a scalar register)
  const float unit = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(
      EPI == kBf16 ? unit_of(g.up, g.over) : EPI == kGrad && g.grad ? *g.up : 1.0f)));
  Copies<T, TA> ca;
  Copies<T, TB> cb;
  ca.init(wave, lane, g.lda);
  cb.init(wave, lane, g.ldb);
  const uint32_t lds0 = lds_offset(lds);
  auto copy_stage = [&](const Unit& u, int t, int buf) {
    const uint32_t to = lds0 + uint32_t(buf) * S::STAGE + uint32_t(wave) * 4096;
    const int k = u.k0 + t * kStageK;
    ca.issue(g.a, g.lda, u.m0, g.m, k, u.k1, to);
    cb.issue(g.b, g.ldb, u.n0, g.n, k, u.k1, to + S::OPERAND);
  };

  // operand reads: block x of 32 rows (columns), k step s of 16
  const int swz = (col >> 1) & 7;
  const int grp = (lane >> 4) & 1, i16 = lane & 15;
  auto read_rows = [&](const uint8_t* base, int x, int s) {
    return read16(base + (32 * x + col) * 128 + (((2 * s + half) ^ swz) << 4));
  };
  auto read_of_k = [&](const uint8_t* base, int x, int s) {
    const int row = 16 * s + 8 * half + (i16 >> 2);
    const int chunk = (4 * x + 2 * grp + ((i16 & 3) >> 1)) ^ (4 * (i16 >> 2));
    const uint8_t* p = base + row * (2 * T) + chunk * 16 + (i16 & 1) * 8;
    return read_transposed(p, p + 4 * (2 * T));
  };
  struct Frags {
    v8bf a[2][S::MB], b[2][S::NB];
  };
  auto read_half = [&](Frags& f, int buf, int h) {
    const uint8_t* st = lds + buf * S::STAGE;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int x = 0; x < S::MB; ++x)
        f.a[s][x] = TA ? read_of_k(st, wm * S::MB + x, 2 * h + s)
                       : read_rows(st, wm * S::MB + x, 2 * h + s);
#pragma unroll
      for (int x = 0; x < S::NB; ++x)
        f.b[s][x] = TB ? read_of_k(st + S::OPERAND, wn * S::NB + x, 2 * h + s)
                       : read_rows(st + S::OPERAND, wn * S::NB + x, 2 * h + s);
    }
  };
  v16f acc[S::MB][S::NB];
  auto clear = [&]() {
#pragma unroll
    for (int x = 0; x < S::MB; ++x)
#pragma unroll
      for (int y = 0; y < S::NB; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
  };
  auto multiply = [&](const Frags& f, int s) {
#pragma unroll
    for (int x = 0; x < S::MB; ++x)
#pragma unroll
      for (int y = 0; y < S::NB; ++y) acc[x][y] = mfma(f.a[s][x], f.b[s][y], acc[x][y]);
  };
  // (keeps the products where they stand, ahead of the barrier and copies that
  // follow)
  auto pin = [&]() {
#pragma unroll
    for (int x = 0; x < S::MB; ++x)
#pragma unroll
      for (int y = 0; y < S::NB; ++y) {
        // (where a wave has 512 registers its accumulators lie in the second half)
        if constexpr (T == 256 || ST == 2) asm volatile("" : "+v"(acc[x][y]));
        else asm volatile("" : "+a"(acc[x][y]));
      }
  };

  // ---- what the epilogue takes of the wave's 64 tokens (the loss's products): target,
  // lse and gradient, brought into the wave's own LDS with the tile's first stages
  // (loaded in the epilogue, each wait for them would wait for the next tile's copies)
  constexpr int TAKEN = EPI == kGrad ? 5 : STATS ? 2 : 0;
  const int mw = wm * S::MB * 32, nw = wn * 64;
  auto take = [&](const Unit& u) {
    if constexpr (MANY && TAKEN > 0) {
      const int n = u.n0 + nw, there = min(max(g.n - n, 0), 64);
      const uint32_t to = lds_offset(own), lane4 = uint32_t(lane) * 4;
      const v4i t = make_rsrc(g.targets + n, uint32_t(there) * 8);
      copy4(t, 2 * lane4, to);
      copy4(t, 2 * lane4 + 4, to + 256);
      if constexpr (EPI == kGrad) {
        copy4(make_rsrc(g.lse + n, uint32_t(there) * 4), lane4, to + 512);
        copy4(make_rsrc(g.grad + n, g.grad ? uint32_t(there) * 4 : 0u), lane4, to + 768);
        copy4(make_rsrc(g.losses + n, g.losses ? uint32_t(there) * 4 : 0u), lane4, to + 1024);
      }
    }
  };
  struct Token {
    int64_t target;
    float lse, grad, loss;
  };
  auto token_of = [&](const Unit& u, int y, int col) {  // (of a row past the tokens: anything)
    Token t{};
    if constexpr (MANY) {
      const uint8_t* p = own + (32 * y + col) * 4;
      t.target = int64_t(uint64_t(*reinterpret_cast<const uint32_t*>(p)) |
                         uint64_t(*reinterpret_cast<const uint32_t*>(p + 256)) << 32);
      if constexpr (EPI == kGrad) {
        t.lse = *reinterpret_cast<const float*>(p + 512);
        t.grad = g.grad ? *reinterpret_cast<const float*>(p + 768) : 1.0f;
        t.loss = *reinterpret_cast<const float*>(p + 1024);
      }
    } else {
      const int64_t n = min(u.n0 + nw + 32 * y + col, g.n - 1);
      t.target = g.targets[n];
      if constexpr (EPI == kGrad) {
        t.lse = g.lse[n];
        t.grad = g.grad ? g.grad[n] : 1.0f;
        t.loss = g.losses ? g.losses[n] : 0.0f;
      }
    }
    return t;
  };
  // the target's place among the lane's values of the tile, negative if it is not there
  auto place_of = [&](const Unit& u, int64_t target, int half) {
    const int64_t w = target - g.first - u.m0;
    return w >= 0 && w < min(T, g.m - u.m0) ? int(w) - mw - 4 * half : -1;
  };

  // ---- results: acc[x][y][r] is m = mw + 4 half + 32 x + 8 (r / 4) + r % 4, n = nw + 32
  // y + col of the tile
  constexpr int STORES = S::NB * (S::MB / 2) * 4;  // instructions a wave
  // 16-bit values as rows: 32 x 64 at a time through the wave's own LDS, and out in
  // runs of 128 bytes (all instructions are issued, so that they can be counted)
  auto store_rows = [&](const Unit& u, int cols, int lane, auto value) {
    const int col = lane & 31, half = lane >> 5, swz = (col >> 1) & 7;
    const int64_t row = g.ldo * 2;
    const int rows = min(g.n - u.n0 - nw, 64);
    const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
        static_cast<uint16_t*>(g.out) + int64_t(u.n0 + nw) * g.ldo + u.m0, 0,
        rows > 0 ? int(uint32_t((rows - 1) * row) + uint32_t(cols - u.m0) * 2) : 0, 0x00020000);
#pragma unroll
    for (int y = 0; y < S::NB; ++y)
#pragma unroll
      for (int xp = 0; xp < S::MB / 2; ++xp) {
#pragma unroll
        for (int x = 2 * xp; x < 2 * xp + 2; ++x)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = 4 * (x & 1) + q;
            *reinterpret_cast<uint2*>(own + col * 128 + ((c ^ swz) << 4) + half * 8) =
                value(x, y, q);
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 3), c = lane & 7;
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          const u4 w = *reinterpret_cast<const u4*>(own + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
          const int m = mw + 64 * xp + 8 * c;
          const uint32_t at = u.m0 + m < cols ? uint32_t((32 * y + r) * row) + uint32_t(m) * 2
                                              : kOutOfRange;
          __builtin_amdgcn_raw_buffer_store_b128(w, out, at, 0, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
  };
  auto finish = [&](const Unit& u) {
    // (what it derives from the lane is not kept through the products)
    const int lane = fresh(threadIdx.x & 63), col = lane & 31, half = lane >> 5;
    // classes of the lane's part of the tile, behind whose end are zeros
    const int there = g.m - u.m0 - mw - 4 * half;
    if constexpr (EPI == kFp32) {
      float* out = static_cast<float*>(g.out) + int64_t(u.split) * g.split_stride;
#pragma unroll
      for (int y = 0; y < S::NB; ++y) {
        const int n = u.n0 + nw + 32 * y + col;
        if (n >= g.n) continue;
#pragma unroll
        for (int x = 0; x < S::MB; ++x)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int m = u.m0 + mw + 4 * half + 32 * x + 8 * q;
            if (m >= g.m) continue;
            float4* p = reinterpret_cast<float4*>(out + int64_t(n) * g.ldo + m);
            float4 v = make_float4(acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2],
                                   acc[x][y][4 * q + 3]);
            if (g.add) {
              const float4 o = *p;
              v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            *p = v;
          }
      }
    }
    if constexpr (EPI == kBf16)
      store_rows(u, g.m, lane, [&](int x, int y, int q) {
        const v16f& e = acc[x][y];
        return make_uint2(pack2(e[4 * q] * unit, e[4 * q + 1] * unit),
                          pack2(e[4 * q + 2] * unit, e[4 * q + 3] * unit));
      });
    if constexpr (EPI == kGrad) {
      // (of g and the exponentials whole tiles are written: what lies behind the classes
      // is zero)
      // (a target's is its p times `of_p`, plus less[])
      const float of_p = g.losses ? 0.0f : 1.0f;
      float off[2], scale[2], less[2];
      int rel[2];
      bool keep[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const Token t = token_of(u, y, col);
        keep[y] = t.target != g.ignore;
        rel[y] = place_of(u, t.target, half);
        scale[y] = g.grad ? t.grad / unit : 1.0f;
        // (a target outside the vocabulary has a loss that is NaN, and so are its
        // gradients)
        if (t.target < 0 || t.target >= g.classes) scale[y] = NAN;
        off[y] = t.lse * kLog2e;
        less[y] = g.losses ? less_one(t.loss) : -1.0f;
      }
      store_rows(u, u.m0 + T, lane, [&](int x, int y, int q) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2_fast(__builtin_fmaf(acc[x][y][4 * q + r], kLog2e, -off[y]));
          const float at = rel[y] == 32 * x + 8 * q + r ? __builtin_fmaf(p, of_p, less[y]) : p;
          v[r] = keep[y] ? at * scale[y] : 0.0f;
        }
        if (u.m0 + T > g.m) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            v[r] = __int_as_float(__float_as_int(v[r]) & ((32 * x + 8 * q + r - there) >> 31));
        }
        return make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
      });
    }
    if constexpr (STATS) {
      // maxima and sums of the two waves along m meet in their own LDS, [64] each
      float* const mine = reinterpret_cast<float*>(own + 1024);
      const float* const other =
          reinterpret_cast<const float*>(spare + (wave ^ 1) * PRIVATE + 1024);
      int rel[2];
#pragma unroll
      for (int y = 0; y < S::NB; ++y) rel[y] = place_of(u, token_of(u, y, col).target, half);
#pragma unroll
      for (int y = 0; y < S::NB; ++y) {
        const int n = u.n0 + nw + 32 * y + col;
        const bool here = n < g.n && rel[y] >= 0 && rel[y] < 32 * S::MB && (rel[y] & 4) == 0;
        if (__ballot(here)) {  // (few of the tiles hold a target of theirs)
          // 32 x 32 values through the wave's LDS, where a lane can pick
          float* const at = reinterpret_cast<float*>(own) + col * 32 + 4 * half;
#pragma unroll
          for (int x = 0; x < S::MB; ++x) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(at + 8 * q) =
                  make_float4(acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2],
                              acc[x][y][4 * q + 3]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (here && rel[y] >> 5 == x) g.picked[n] = at[rel[y] & 31];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
      }
#pragma unroll
      for (int y = 0; y < S::NB; ++y) {
        float top = -INFINITY;
        if (u.m0 + T > g.m) {
#pragma unroll
          for (int x = 0; x < S::MB; ++x) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              acc[x][y][r] = 32 * x + 8 * (r >> 2) + (r & 3) < there ? acc[x][y][r] : -INFINITY;
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int x = 0; x < S::MB; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[x][y][r]);
        top = fmaxf(top, __shfl_xor(top, 32));
        if (half == 0) mine[32 * y + col] = top;
      }
      sync_lds();
#pragma unroll
      for (int y = 0; y < S::NB; ++y) {
        const float top = fmaxf(mine[32 * y + col], other[32 * y + col]);
        const float off = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < S::MB; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = exp2_fast((acc[x][y][r] - off) * kLog2e);
            sum += e;
            if constexpr (EPI == kExps) acc[x][y][r] = e;
          }
        sum += __shfl_xor(sum, 32);
        if (half == 0) mine[64 + 32 * y + col] = sum;
      }
      sync_lds();
      const int n = u.n0 + nw + lane;
      if (wm == 0 && n < g.n) {
        const float top = fmaxf(mine[lane], other[lane]);
        g.part[int64_t(u.m0 / T) * g.n + n] =
            make_float2(top == -INFINITY ? 0.0f : top, mine[64 + lane] + other[64 + lane]);
      }
      if constexpr (EPI == kExps) {
        sync_lds();
        store_rows(u, u.m0 + T, lane, [&](int x, int y, int q) {
          const v16f& e = acc[x][y];
          return make_uint2(half2(e[4 * q] * kExpsUp, e[4 * q + 1] * kExpsUp),
                            half2(e[4 * q + 2] * kExpsUp, e[4 * q + 3] * kExpsUp));
        });
      }
    }
  };

  Unit u = unit_at<T>(g, int(blockIdx.x));
  Frags f0, f1;
  clear();
  if constexpr (MANY) {
    const int units = g.tiles_m * g.tiles_n * g.splits;
    // instructions in flight behind a tile's second stage: the result's stores (at
    // least), and what the next epilogue takes
    constexpr int BEHIND = (EPI == kBf16 || EPI == kGrad || EPI == kExps ? STORES : 0) + TAKEN;
    copy_stage(u, 0, 0);
    copy_stage(u, 1, 1);
    take(u);
    wait_and_sync<8 + TAKEN>();
    read_half(f0, 0, 0);
    int buf = 0;
    for (int at = int(blockIdx.x); at < units; at += int(gridDim.x)) {
      const bool more = at + int(gridDim.x) < units;
      Unit next = u;
      if (more) next = unit_at<T>(g, at + int(gridDim.x));
      else next.k1 = next.k0;  // (copies read nothing)
      for (int t = 0; t < u.stages; ++t, buf ^= 1) {
        read_half(f1, buf, 1);
        multiply(f0, 0);
        pin();
        if (t == 0 && at >= int(gridDim.x)) wait_and_sync<BEHIND>();
        else wait_and_sync<0>();
        multiply(f0, 1);
        pin();
        __builtin_amdgcn_sched_barrier(0);
        const bool last = t + 2 >= u.stages;
        copy_stage(last ? next : u, last ? t + 2 - u.stages : t + 2, buf);
        __builtin_amdgcn_sched_barrier(0);
        // (after the last stage: the next tile's first one)
        read_half(f0, buf ^ 1, 0);
        multiply(f1, 0);
        multiply(f1, 1);
      }
      finish(u);
      clear();
      u = next;
      if (more) take(u);
    }
    // (copies still in flight read nothing, but write zeros)
    wait_and_sync<0>();
  } else {
    // (copies past the last stage read nothing and keep the count of what is in flight)
    constexpr int kAhead = 8 * (S::STAGES - 2);
#pragma unroll
    for (int t = 0; t < S::STAGES - 1; ++t) copy_stage(u, t, t);
    wait_and_sync<kAhead>();
    copy_stage(u, S::STAGES - 1, S::STAGES - 1);
    read_half(f0, 0, 0);
    for (int t = 0; t < u.stages; ++t) {
      read_half(f1, t % S::STAGES, 1);
      multiply(f0, 0);
      pin();
      wait_and_sync<kAhead>();
      multiply(f0, 1);
      pin();
      __builtin_amdgcn_sched_barrier(0);
      copy_stage(u, t + S::STAGES, t % S::STAGES);
      __builtin_amdgcn_sched_barrier(0);
      read_half(f0, (t + 1) % S::STAGES, 0);
      multiply(f1, 0);
      multiply(f1, 1);
    }
    wait_and_sync<0>();
    finish(u);
  }
}

// ---- the joins ----------------------------------------------------------------

// Every token's lse and loss from its partial maxima and sums: 32 tokens a block, 32
// threads each, and the block's sum of losses and tokens that count into sums.  With
// `done`, the counter that the launch before cleared, the block that is last adds up
// all of them: a launch less, but every block publishes its sums past its XCD's L2
// (4096 tokens in 512 blocks: 15 us against 4), so for few blocks only.
constexpr int kJoinTokens = 32, kJoinThreads = 32 * kJoinTokens, kJoinLast = 32;

// The losses' sum or mean, and the tokens that count, from n blocks' sums, in one
// order.
template <typename Load>
TCFP_DEV void add_up(int n, int mean, Load load, float* total, float* count) {
  __shared__ double2 d[256];
  const int t = threadIdx.x;
  if (t < 256) {
    double a = 0.0, b = 0.0;
    for (int i = t; i < n; i += 256) a += load(2 * i), b += load(2 * i + 1);
    d[t] = make_double2(a, b);
  }
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (t < o) d[t].x += d[t + o].x, d[t].y += d[t + o].y;
    __syncthreads();
  }
  if (t == 0) {
    *total = float(mean ? d[0].x / d[0].y : d[0].x);
    *count = float(d[0].y);
  }
}
__global__ __launch_bounds__(256) void total_loss_kernel(const double* __restrict__ sums, int n,
                                                         int mean, float* total, float* count) {
  add_up(n, mean, [&](int i) { return sums[i]; }, total, count);
}

__global__ __launch_bounds__(kJoinThreads) void join_losses_kernel(
    const float2* __restrict__ part, int parts, const float* __restrict__ picked,
    const int64_t* __restrict__ targets, int64_t ignore, int64_t classes, int tokens,
    float* __restrict__ losses, float* __restrict__ lse, double* sums, int* done, int mean,
    float* total, float* count_out) {
  __shared__ float2 s[32][kJoinTokens];
  __shared__ bool last;
  const int tl = threadIdx.x % kJoinTokens, slice = threadIdx.x / kJoinTokens;
  const int t = int(blockIdx.x) * kJoinTokens + tl;
  float top = -INFINITY, sum = 0.0f;
  auto add = [&](const float2& p) {
    if (p.y == 0.0f) return;
    const float next = fmaxf(top, p.x);
    sum = (sum == 0.0f ? 0.0f : sum * exp2_fast((top - next) * kLog2e)) +
          p.y * exp2_fast((p.x - next) * kLog2e);
    top = next;
  };
  if (t < tokens)
    for (int i = slice; i < parts; i += 4 * 32) {
      float2 p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[j] = i + 32 * j < parts ? part[int64_t(i + 32 * j) * tokens + t]
                                  : make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) add(p[j]);
    }
  s[slice][tl] = make_float2(top, sum);
  __syncthreads();
  double loss = 0.0, count = 0.0;
  if (slice == 0 && t < tokens) {
    for (int i = 1; i < 32; ++i) add(s[i][tl]);
    const float rest = log2_fast(sum) * kLn2;
    const int64_t target = targets[t];
    const bool keep = target != ignore;
    const float each = !keep ? 0.0f : target < 0 || target >= classes
                                     ? NAN : (top - picked[t]) + rest;
    lse[t] = top + rest;
    losses[t] = each;
    loss = each;
    count = keep ? 1.0 : 0.0;
  }
  if (!sums) return;
  if (threadIdx.x < 64) {  // (the block's tokens are its first 32 threads)
#pragma unroll
    for (int o = kJoinTokens / 2; o > 0; o >>= 1) {
      loss += __shfl_xor(loss, o);
      count += __shfl_xor(count, o);
    }
    if (threadIdx.x == 0 && !done) {
      sums[2 * blockIdx.x] = loss;
      sums[2 * blockIdx.x + 1] = count;
    } else if (threadIdx.x == 0) {
      __hip_atomic_store(sums + 2 * blockIdx.x, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * blockIdx.x + 1, count, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             int(gridDim.x) - 1;
    }
  }
  if (!done) return;
  __syncthreads();
  if (!last) return;
  add_up(int(gridDim.x), mean,
         [&](int i) {
           return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
         },
         total, count_out);
}

// The total of no tokens.
__global__ void no_tokens_kernel(int mean, float* total, float* count) {
  *total = mean ? NAN : 0.0f;
  *count = 0.0f;
}

// The exponentials of tokens x classes (fp16, rows ld apart, kExpsUp times those relative
// to the maxima of their tiles) turned into g (bf16) in place, eight a thread.
template <int T>
__global__ __launch_bounds__(256) void exps_to_grad_kernel(
    uint16_t* __restrict__ x, int64_t ld, const float2* __restrict__ part,
    const float* __restrict__ lse, const float* __restrict__ losses,
    const int64_t* __restrict__ targets, int64_t ignore, int64_t classes, int tokens) {
  const int t = int(blockIdx.y) * 8 + threadIdx.x / 32;
  if (t >= tokens) return;
  const int64_t target = targets[t];
  const bool keep = target != ignore;
  const float c = target < 0 || target >= classes ? NAN : 1.0f;  // (as its loss)
  const float l = lse[t], less = less_one(losses[t]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t v0 = (int64_t(blockIdx.x) * 128 + i * 32 + threadIdx.x % 32) * 8;
    if (v0 >= classes) return;
    const float f = exp2_fast((part[v0 / T * tokens + t].x - l) * kLog2e) * (c / kExpsUp);
    uint4* p = reinterpret_cast<uint4*>(x + int64_t(t) * ld + v0);
    typedef _Float16 v8h __attribute__((ext_vector_type(8)));
    const v8h e = __builtin_bit_cast(v8h, *p);
    const int at = target >= v0 && target < v0 + 8 ? int(target - v0) : -1;
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // (what lies behind the classes stays zero)
      const float z = v0 + j < classes ? (j == at ? less : float(e[j]) * f) : 0.0f;
      g[j] = keep ? z : 0.0f;
    }
    *p = make_uint4(pack2(g[0], g[1]), pack2(g[2], g[3]), pack2(g[4], g[5]), pack2(g[6], g[7]));
  }
}

// Two arrays of bf16, eights of them, times *by, in place; nothing is to be done
// for 1, what the gradient of a loss is most of the time.
__global__ __launch_bounds__(256) void scale_kernel(uint16_t* a, int64_t a_eights, uint16_t* b,
                                                    int64_t b_eights, const float* by) {
  const float f = *by;
  if (f == 1.0f) return;
  const int64_t step = int64_t(gridDim.x) * 256;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < a_eights + b_eights; i += step) {
    uint4* p = i < a_eights ? reinterpret_cast<uint4*>(a) + i
                            : reinterpret_cast<uint4*>(b) + (i - a_eights);
    const uint4 x = *p;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      y[j] = pack2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xFFFF0000u) * f);
    *p = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// The largest of the tokens' gradients that is finite; 1 if that is 0.  What a token that
// is left out has does not count: divided by it, the others' could fall below bf16's
// smallest values.
__global__ __launch_bounds__(1024) void largest_kernel(const float* __restrict__ grad,
                                                       const int64_t* __restrict__ targets,
                                                       int64_t ignore, int64_t classes, int tokens,
                                                       float* unit) {
  __shared__ float s[16];
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < tokens; i += 1024) {
    const float x = fabsf(grad[i]);
    const int64_t target = targets[i];
    if (x < INFINITY && target != ignore && target >= 0 && target < classes) top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
  *unit = top == 0.0f ? 1.0f : top;
}

// out = the sum of `splits` fp32 [n, m] arrays times unit in bf16, in order; eight
// columns a thread.
__global__ __launch_bounds__(256) void round_sum_kernel(const float* __restrict__ part, int splits,
                                                        int64_t stride, int64_t eights,
                                                        const float* up, const float* over,
                                                        uint16_t* __restrict__ out) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= eights) return;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4* p = reinterpret_cast<const float4*>(part + s * stride) + 2 * i;
    const float4 a = p[0], b = p[1];
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  const float unit = unit_of(up, over);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= unit;
  reinterpret_cast<uint4*>(out)[i] =
      make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}

// ---- plans ----------------------------------------------------------------------

constexpr int kCus = 256;
// g of a run of classes takes at most this much of the workspace, but for runs
// of 256 classes, the shortest: 512 bytes a token.
constexpr int64_t kRunBytes = int64_t(256) << 20;
// What g of all classes may take where the forward makes the gradients.
constexpr int64_t kTrainBytes = int64_t(1) << 30;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int launch_status() { return hipGetLastError() == hipSuccess ? TCFP_OK : TCFP_ERR_HIP; }

// How C [n, m] over k is computed: tile, stages in LDS, splits of k.
struct Cut {
  int tile, ring, splits, k_run;
};
// What `units` tiles of `stages` each take, us, by what was measured: a stage 1.5,
// 0.55 and (two workgroups on a CU) 0.98 us, first loads and result 9.5, 4 and 5; e.g.
// 2048 x 8192 over 4096: 107 us in tiles of 256, 125 with 128 and two stages, 150
// with four; 64 x 32768 over 4096, where W comes from HBM: 55 with 128 and four
// stages, 73 with two; 1000 x 8192 over 1056: 28 with two, 33 with four.
double cost(int tile, int ring, int64_t units, int64_t stages) {
  if (tile == 256)
    return double(ceil_div(units, kCus)) * (std::max(1.5 * double(stages), 4.0) + 9.5);
  if (ring == 4) return double(ceil_div(units, kCus)) * (0.55 * double(stages) + 4);
  const int64_t rounds = units / (2 * kCus), rest = units - rounds * 2 * kCus;
  return double(rounds) * (0.98 * double(stages) + 5) +
         (rest > kCus ? 0.98 * double(stages) + 5 : rest > 0 ? 0.7 * double(stages) + 4 : 0.0);
}
// Splits write fp32 parts, 3.5 TB/s with their sum, and take a launch more.
Cut cut_of(int64_t n, int64_t m, int64_t k, bool may_split) {
  const int64_t stages = std::max<int64_t>(ceil_div(k, kStageK), 1);
  Cut best{};
  double least = INFINITY;
  for (const auto& [tile, ring] : {std::pair<int, int>{256, 2}, {128, 2}, {128, 4}}) {
    const int64_t tiles = ceil_div(n, tile) * ceil_div(m, tile);
    for (int64_t s = 1; s <= (may_split ? std::min<int64_t>(64, stages) : 1); ++s) {
      if (s > 1 && tiles * s > 2 * kCus) break;
      const int64_t each = ceil_div(stages, s);
      const double t = cost(tile, ring, tiles * s, each) +
                       (s > 1 ? double(n) * double(m) * 8 * double(s) / 3.5e6 + 4 : 0.0);
      if (t < least) {
        least = t;
        best = {tile, ring, int(ceil_div(stages, each)), int(each * kStageK)};
      }
    }
  }
  return best;
}
Cut logits_cut(int64_t tokens, int64_t classes, int64_t dim) {
  return cut_of(tokens, classes, dim, false);
}
// Classes of a run of the backward pass (a multiple of 256, whole tiles).
int64_t run_of(int64_t tokens, int64_t vocab) {
  // (rows of a run stay within a descriptor's reach)
  const int64_t most = std::clamp<int64_t>(
      kRunBytes / (2 * std::max<int64_t>(tokens, 1)) / 256, 1, 4096) * 256;
  const int64_t all = ceil_div(vocab, 256) * 256;
  const int64_t runs = ceil_div(all, most);
  return ceil_div(ceil_div(all, runs), 256) * 256;
}

template <int T, int ST, bool TA, bool TB, int EPI>
int launch(Product p, hipStream_t st) {
  constexpr int THREADS = Shape<T, ST>::THREADS;
  p.tiles_m = int(ceil_div(p.m, T));
  p.tiles_n = int(ceil_div(p.n, T));
  const int64_t units = int64_t(p.tiles_m) * p.tiles_n * p.splits;
  if (!grid_x_fits(units, THREADS) || units > INT32_MAX) return TCFP_ERR_SHAPE;
  // (tiles of 256: a workgroup a CU, which takes several)
  const unsigned grid = unsigned(T == 256 ? std::min<int64_t>(units, kCus) : units);
  product_kernel<T, ST, TA, TB, EPI><<<grid, THREADS, 0, st>>>(p);
  return launch_status();
}
template <bool TA, bool TB, int EPI>
int launch_cut(const Cut& c, Product p, hipStream_t st) {
  p.splits = c.splits;
  p.k_run = c.k_run;
  return c.tile == 256 ? launch<256, 2, TA, TB, EPI>(p, st)
         : c.ring == 2 ? launch<128, 2, TA, TB, EPI>(p, st)
                       : launch<128, 4, TA, TB, EPI>(p, st);
}

struct Layout {
  int64_t run;      // classes
  Cut dh, dw;
  size_t g, sum_h, sum_w;  // bytes: g of a run, fp32 sums of dh and of dW
};
Layout layout_of(int64_t tokens, int64_t vocab, int64_t dim, bool need_h, bool need_w) {
  Layout l{};
  l.run = run_of(tokens, vocab);
  l.g = align256(size_t(tokens) * size_t(l.run) * 2);
  if (need_h) {
    l.dh = cut_of(tokens, dim, std::min(l.run, vocab), true);
    if (l.dh.splits > 1 || l.run < vocab)
      l.sum_h = align256(size_t(l.dh.splits) * size_t(tokens) * size_t(dim) * 4);
  }
  if (need_w) {
    l.dw = cut_of(std::min(l.run, vocab), dim, tokens, true);
    if (l.dw.splits > 1)
      l.sum_w = align256(size_t(l.dw.splits) * size_t(std::min(l.run, vocab)) * size_t(dim) * 4);
  }
  return l;
}

int check_sizes(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int64_t tokens,
                int64_t vocab, int64_t dim) {
  if (tokens < 0 || vocab < 1 || dim < 8 || dim % 8 || tokens > INT32_MAX / 2 ||
      vocab > INT32_MAX / 2 || dim > INT32_MAX / 2 || ldh < dim || ldw < dim)
    return TCFP_ERR_SHAPE;
  // (32-bit offsets within a tile's rows)
  if (256 * ldh * 2 + dim * 2 >= kMaxSpan || 256 * ldw * 2 + dim * 2 >= kMaxSpan)
    return TCFP_ERR_SHAPE;
  if (!aligned16(hidden) || !aligned16(weight) || ldh % 8 || ldw % 8) return TCFP_ERR_ALIGN;
  return TCFP_OK;
}

// The workspace of one pass over all classes at once.
Layout train_layout(int64_t tokens, int64_t vocab, int64_t dim, bool need_h, bool need_w) {
  Layout l{};
  l.run = ceil_div(vocab, 256) * 256;
  l.g = align256(size_t(tokens) * size_t(l.run) * 2);
  if (need_h) {
    l.dh = cut_of(tokens, dim, vocab, true);
    if (l.dh.splits > 1) l.sum_h = align256(size_t(l.dh.splits) * size_t(tokens) * size_t(dim) * 4);
  }
  if (need_w) {
    l.dw = cut_of(vocab, dim, tokens, true);
    if (l.dw.splits > 1) l.sum_w = align256(size_t(l.dw.splits) * size_t(vocab) * size_t(dim) * 4);
  }
  return l;
}

struct Head {
  const void* hidden;
  int64_t ldh;
  const void* weight;
  int64_t ldw;
  const int64_t* targets;
  int64_t ignore, tokens, vocab, dim;
};
// z of the classes [v0, v0 + classes).
Product head_product(const Head& h, int64_t v0, int64_t classes) {
  Product p{};
  p.a = static_cast<const uint16_t*>(h.weight) + v0 * h.ldw;
  p.b = static_cast<const uint16_t*>(h.hidden);
  p.lda = h.ldw;
  p.ldb = h.ldh;
  p.m = int(classes);
  p.n = int(h.tokens);
  p.k = int(h.dim);
  p.targets = h.targets;
  p.ignore = h.ignore;
  p.first = v0;
  p.classes = h.vocab;
  return p;
}

// Workspace of losses_of(): parts, the targets' logits, sums of blocks, a counter.
size_t parts_bytes(int64_t tokens, int64_t vocab, int64_t dim) {
  const int64_t parts = ceil_div(vocab, logits_cut(tokens, vocab, dim).tile);
  return align256(size_t(parts) * size_t(tokens) * 8) + align256(size_t(tokens) * 4) +
         align256(size_t(ceil_div(tokens, kJoinTokens)) * 16) + 256;
}
// Losses, and with exps (rows ld apart) what exps_to_grad_kernel takes.
int losses_of(const Head& h, float* losses, float* lse, int mean, float* total, float* count,
              uint8_t* ws, uint16_t* exps, int64_t ld, hipStream_t st) {
  const Cut cut = logits_cut(h.tokens, h.vocab, h.dim);
  const int64_t parts = ceil_div(h.vocab, cut.tile);
  const unsigned blocks = unsigned(ceil_div(h.tokens, kJoinTokens));
  Product p = head_product(h, 0, h.vocab);
  p.out = exps;
  p.ldo = ld;
  p.part = reinterpret_cast<float2*>(ws);
  ws += align256(size_t(parts) * size_t(h.tokens) * 8);
  p.picked = reinterpret_cast<float*>(ws);
  ws += align256(size_t(h.tokens) * 4);
  double* sums = total ? reinterpret_cast<double*>(ws) : nullptr;
  p.done = reinterpret_cast<int*>(ws + align256(size_t(blocks) * 16));
  const bool last = blocks <= kJoinLast;
  if (!grid_x_fits(blocks, kJoinThreads)) return TCFP_ERR_SHAPE;
  const int rc = exps ? launch_cut<false, false, kExps>(cut, p, st)
                      : launch_cut<false, false, kStats>(cut, p, st);
  if (rc != TCFP_OK) return rc;
  join_losses_kernel<<<blocks, kJoinThreads, 0, st>>>(
      p.part, int(parts), p.picked, h.targets, h.ignore, h.vocab, int(h.tokens), losses, lse, sums,
      last && total ? p.done : nullptr, mean, total, count);
  if (total && !last)
    total_loss_kernel<<<1, 256, 0, st>>>(sums, int(blocks), mean, total, count);
  return launch_status();
}

int round_sum(const float* part, int splits, int64_t values, const float* up, const float* over,
              void* out, hipStream_t st) {
  const int64_t eights = values / 8, blocks = ceil_div(eights, 256);
  if (!grid_x_fits(blocks, 256)) return TCFP_ERR_SHAPE;
  round_sum_kernel<<<unsigned(blocks), 256, 0, st>>>(part, splits, values, eights, up, over,
                                                     static_cast<uint16_t*>(out));
  return launch_status();
}

// What g of the classes [v0, v0 + classes) gives: their rows of dW, and their part of
// dh (into sum_h where the layout has it: added up over the runs, and not yet times
// unit).
int products_of(const Head& h, const Layout& l, const uint16_t* g, int64_t v0, int64_t classes,
                const float* up, const float* over, void* grad_hidden, void* grad_weight,
                float* sum_h, float* sum_w, hipStream_t st) {
  if (grad_hidden) {
    // dh[t][d] += sum over the classes of g[t][v] W[v][d]
    Product q{};
    q.a = static_cast<const uint16_t*>(h.weight) + v0 * h.ldw;
    q.b = g;
    q.lda = h.ldw;
    q.ldb = l.run;
    q.m = int(h.dim);
    q.n = int(h.tokens);
    q.k = int(classes);
    q.ldo = h.dim;
    int done;
    if (l.sum_h) {
      q.out = sum_h;
      q.split_stride = h.tokens * h.dim;
      q.add = v0 > 0;
      // (a last, shorter run may leave splits without classes: nothing to add)
      Cut cut = l.dh;
      if (v0 > 0) cut.splits = int(std::min<int64_t>(cut.splits, ceil_div(classes, cut.k_run)));
      done = launch_cut<true, false, kFp32>(cut, q, st);
    } else {
      q.out = grad_hidden;
      q.up = up;
      q.over = over;
      done = launch_cut<true, false, kBf16>(l.dh, q, st);
    }
    if (done != TCFP_OK) return done;
  }
  if (!grad_weight) return TCFP_OK;
  // dW[v][d] = sum over tokens of g[t][v] h[t][d]
  Product q{};
  q.a = static_cast<const uint16_t*>(h.hidden);
  q.b = g;
  q.lda = h.ldh;
  q.ldb = l.run;
  q.m = int(h.dim);
  q.n = int(classes);
  q.k = int(h.tokens);
  q.ldo = h.dim;
  uint16_t* out = static_cast<uint16_t*>(grad_weight) + v0 * h.dim;
  if (l.dw.splits == 1) {
    q.out = out;
    q.up = up;
    q.over = over;
    return launch_cut<true, true, kBf16>(l.dw, q, st);
  }
  q.out = sum_w;
  q.split_stride = classes * h.dim;
  const int done = launch_cut<true, true, kFp32>(l.dw, q, st);
  return done != TCFP_OK
             ? done
             : round_sum(sum_w, l.dw.splits, classes * h.dim, up, over, out, st);
}

}  // namespace

extern "C" {

size_t tcfp_linear_cross_entropy_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim) {
  if (tokens <= 0 || vocab <= 0 || dim <= 0) return 0;
  return parts_bytes(tokens, vocab, dim);
}

int tcfp_linear_cross_entropy(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                              const int64_t* targets, int64_t ignore, int64_t tokens,
                              int64_t vocab, int64_t dim, float* losses, float* lse, int mean,
                              float* total, float* count, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const int rc = check_sizes(hidden, ldh, weight, ldw, tokens, vocab, dim);
  if (rc != TCFP_OK) return rc;
  if (!total != !count) return TCFP_ERR_SHAPE;
  const auto st = static_cast<hipStream_t>(stream);
  if (tokens == 0) {
    if (total) no_tokens_kernel<<<1, 1, 0, st>>>(mean, total, count);
    return launch_status();
  }
  if (!workspace || workspace_bytes < parts_bytes(tokens, vocab, dim) || !aligned16(workspace))
    return TCFP_ERR_WORKSPACE;
  return losses_of({hidden, ldh, weight, ldw, targets, ignore, tokens, vocab, dim}, losses, lse,
                   mean, total, count, static_cast<uint8_t*>(workspace), nullptr, 0, st);
}

size_t tcfp_linear_cross_entropy_train_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim,
                                                       int need_hidden, int need_weight) {
  // (the second and third: the grid of the pass over g, a descriptor's reach)
  if (tokens <= 0 || vocab <= 0 || dim <= 0 || tokens > 65535 * 8 || vocab > 1 << 20) return 0;
  const Layout l = train_layout(tokens, vocab, dim, need_hidden != 0, need_weight != 0);
  if (int64_t(l.g) > kTrainBytes) return 0;
  return l.g + l.sum_h + l.sum_w + parts_bytes(tokens, vocab, dim);
}

int tcfp_linear_cross_entropy_train(const void* hidden, int64_t ldh, const void* weight,
                                    int64_t ldw, const int64_t* targets, int64_t ignore,
                                    int64_t tokens, int64_t vocab, int64_t dim, float* losses,
                                    float* lse, int mean, float* total, float* count,
                                    void* grad_hidden, void* grad_weight, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const int rc = check_sizes(hidden, ldh, weight, ldw, tokens, vocab, dim);
  if (rc != TCFP_OK) return rc;
  if (!aligned16(grad_hidden) || !aligned16(grad_weight)) return TCFP_ERR_ALIGN;
  const bool need_h = grad_hidden != nullptr, need_w = grad_weight != nullptr;
  const size_t need =
      tcfp_linear_cross_entropy_train_workspace_bytes(tokens, vocab, dim, need_h, need_w);
  if (need == 0 || !total || !count) return TCFP_ERR_SHAPE;
  if (!workspace || workspace_bytes < need || !aligned16(workspace)) return TCFP_ERR_WORKSPACE;
  const auto st = static_cast<hipStream_t>(stream);
  const Head head{hidden, ldh, weight, ldw, targets, ignore, tokens, vocab, dim};
  const Layout l = train_layout(tokens, vocab, dim, need_h, need_w);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint16_t* g = reinterpret_cast<uint16_t*>(ws);
  uint8_t* parts = ws + l.g + l.sum_h + l.sum_w;
  int done = losses_of(head, losses, lse, mean, total, count, parts, g, l.run, st);
  if (done != TCFP_OK) return done;
  const dim3 grid(unsigned(ceil_div(vocab, 1024)), unsigned(ceil_div(tokens, 8)));
  const auto* part = reinterpret_cast<const float2*>(parts);
  const float* each = mean ? count : nullptr;
  if (logits_cut(tokens, vocab, dim).tile == 256)
    exps_to_grad_kernel<256><<<grid, 256, 0, st>>>(g, l.run, part, lse, losses, targets, ignore,
                                                   vocab, int(tokens));
  else
    exps_to_grad_kernel<128><<<grid, 256, 0, st>>>(g, l.run, part, lse, losses, targets, ignore,
                                                   vocab, int(tokens));
  if (launch_status() != TCFP_OK) return TCFP_ERR_HIP;
  done = products_of(head, l, g, 0, vocab, nullptr, each, grad_hidden, grad_weight,
                     reinterpret_cast<float*>(ws + l.g),
                     reinterpret_cast<float*>(ws + l.g + l.sum_h), st);
  if (done != TCFP_OK || !l.sum_h) return done;
  return round_sum(reinterpret_cast<float*>(ws + l.g), l.dh.splits, tokens * dim, nullptr, each,
                   grad_hidden, st);
}

int tcfp_scale_bf16(void* a, int64_t a_values, void* b, int64_t b_values, const float* by,
                    void* stream) {
  if (a_values < 0 || b_values < 0 || a_values % 8 || b_values % 8) return TCFP_ERR_SHAPE;
  if (!aligned16(a) || !aligned16(b)) return TCFP_ERR_ALIGN;
  const int64_t eights = (a_values + b_values) / 8;
  if (eights == 0) return TCFP_OK;
  scale_kernel<<<unsigned(std::min<int64_t>(ceil_div(eights, 256), 8 * kCus)), 256, 0,
                 static_cast<hipStream_t>(stream)>>>(static_cast<uint16_t*>(a), a_values / 8,
                                                     static_cast<uint16_t*>(b), b_values / 8, by);
  return launch_status();
}

size_t tcfp_linear_cross_entropy_backward_workspace_bytes(int64_t tokens, int64_t vocab,
                                                          int64_t dim, int need_hidden,
                                                          int need_weight) {
  if (tokens <= 0 || vocab <= 0 || dim <= 0) return 0;
  const Layout l = layout_of(tokens, vocab, dim, need_hidden != 0, need_weight != 0);
  return l.g + l.sum_h + l.sum_w + 256;  // (and unit)
}

int tcfp_linear_cross_entropy_backward(const void* hidden, int64_t ldh, const void* weight,
                                       int64_t ldw, const int64_t* targets, int64_t ignore,
                                       const float* lse, const float* losses, const float* grad,
                                       int64_t grad_step, const float* count, int64_t tokens, int64_t vocab,
                                       int64_t dim, void* grad_hidden, void* grad_weight,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_sizes(hidden, ldh, weight, ldw, tokens, vocab, dim);
  if (rc != TCFP_OK) return rc;
  if (!aligned16(grad_hidden) || !aligned16(grad_weight)) return TCFP_ERR_ALIGN;
  if (grad_step != 0 && grad_step != 1) return TCFP_ERR_SHAPE;
  const bool need_h = grad_hidden != nullptr, need_w = grad_weight != nullptr;
  if (!need_h && !need_w) return TCFP_OK;
  const auto st = static_cast<hipStream_t>(stream);
  if (tokens == 0) {
    if (need_w) {
      const int64_t eights = vocab * dim / 8;
      if (!grid_x_fits(ceil_div(eights, 256), 256)) return TCFP_ERR_SHAPE;
      round_sum_kernel<<<unsigned(ceil_div(eights, 256)), 256, 0, st>>>(
          nullptr, 0, 0, eights, nullptr, nullptr, static_cast<uint16_t*>(grad_weight));
    }
    return launch_status();
  }
  const Layout l = layout_of(tokens, vocab, dim, need_h, need_w);
  if (!workspace || workspace_bytes < l.g + l.sum_h + l.sum_w + 256 || !aligned16(workspace))
    return TCFP_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint16_t* g = reinterpret_cast<uint16_t*>(ws);
  float* sum_h = reinterpret_cast<float*>(ws + l.g);
  float* sum_w = reinterpret_cast<float*>(ws + l.g + l.sum_h);
  const Head head{hidden, ldh, weight, ldw, targets, ignore, tokens, vocab, dim};
  const float* up = grad;
  if (grad_step == 1) {
    float* largest = reinterpret_cast<float*>(ws + l.g + l.sum_h + l.sum_w);
    largest_kernel<<<1, 1024, 0, st>>>(grad, targets, ignore, vocab, int(tokens), largest);
    up = largest;
  }
  for (int64_t v0 = 0; v0 < vocab; v0 += l.run) {
    const int64_t classes = std::min(l.run, vocab - v0);
    Product p = head_product(head, v0, classes);
    p.out = g;
    p.ldo = l.run;
    p.lse = lse;
    p.losses = losses;
    p.grad = grad_step == 1 ? grad : nullptr;
    p.up = up;
    int done = launch_cut<false, false, kGrad>(logits_cut(tokens, classes, dim), p, st);
    if (done == TCFP_OK)
      done = products_of(head, l, g, v0, classes, up, count, grad_hidden, grad_weight, sum_h,
                         sum_w, st);
    if (done != TCFP_OK) return done;
  }
  if (need_h && l.sum_h)
    return round_sum(sum_h, l.dh.splits, tokens * dim, up, count, grad_hidden, st);
  return TCFP_OK;
}

}  // extern "C"
