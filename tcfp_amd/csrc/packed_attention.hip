// Attention within packed sequences, and its gradients (gfx950).
//
//   S = scale Q K^T,  P = softmax(S) over the keys a query sees,  O = P V
//   delta = rowsum(dO * O),  dV = P^T dO,  dS = P * (dO V^T - delta),
//   dQ = scale dS K,  dK = scale dS^T Q
//
// All operands are bf16; scores, maxima, sums, the row statistic L = log2 sum
// 2^S and every accumulator are fp32.  P and dS are rounded to bf16 on their way
// into the second products (2^-8 of each value at most, as the results are rounded
// themselves), of short sequences what dS's rounding left is multiplied too (see
// kShort).  No P is stored: the backward forms it again from L.
//
// Every product runs transposed so that what one leaves in the registers is what
// the next one wants of the lane (the matrix instruction's columns are the
// lanes): forward and dQ have the queries across the lanes, S^T = K Q^T,
// O^T += V^T P^T, dQ^T += K^T dS^T; dK and dV have the keys there, S = Q K^T,
// dV^T += dO^T P, dK^T += Q^T dS.  A row's statistics are then the lane's own, or
// a broadcast.  The order of the eight k that a lane gives an instruction is that
// of its registers, on both sides.  Tiles of the operand that a wave does not keep
// are copied into LDS as they lie and read from there by rows or transposed.
//
// The gradients of K and V are a launch of their own, which forms S and dP again
// (seven products in all instead of five): their sums over the queries then stay
// in registers, in one order, where a single launch would add dQ's or dK's parts
// with atomics.
#include <algorithm>
#include <cmath>

#include "mfma_tiles.h"

using namespace tcfp;

namespace {

constexpr int kStep = 64;  // rows of a tile in LDS
// Where no sequence has more rows than this, dQ and dK take dS as two bf16, its rounding
// and what that left: 1.7e-3 off, as the results' rounding, instead of 2.4e-3 (dV, whose P
// stays one bf16, is 2.3e-3 off either way).  A backward pass takes, with two and with
// one: 32 sequences of 128 tokens, 4 heads of 64, 18.2 us and 17.8, less than its launches
// take the host; 64 of 256, 8 heads of 64, 65 and 61; 256 of 256, 32 / 8 heads of 128, 1490
// and 1326.  Long sequences take the shorter form.
constexpr int kShort = 256;

struct Packed {
  const uint16_t *q, *k, *v, *go;  // [tokens, heads, dim], [keys, kv_heads, dim]
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, go_token, go_head;
  uint16_t* o;            // contiguous: written forward, read backward
  int8_t* low;            // what o's rounding left, see low_part()
  uint16_t *dq, *dk, *dv;  // contiguous
  float* lse;             // [heads, tokens]: log2 of the sum, +inf where nothing is seen
  float* delta;           // [heads, tokens]
  float* part;            // dK and dV of each part in fp32, if there are several
  const int32_t *q_starts, *k_starts;
  int batch, tokens, keys, heads, kv_heads, group;
  float c;      // |scale| * log2(e), 1 for a scale of 0
  float sign;   // of the scale
  float scale;
  int causal, window;
  int tiles;    // of a sequence and head in the launch
  int sets;     // (sequence, K/V head)s
  int parts;    // of a group's heads (dK, dV)
};

// Sequence b: rows of q and of k, and how far its keys reach before its queries.
struct Seq {
  int q0, nq, k0, nk, shift;
};
TCFP_DEV Seq sequence(const Packed& a, int b) {
  Seq s;
  s.q0 = min(max(a.q_starts[b], 0), a.tokens);
  s.nq = max(min(a.q_starts[b + 1], a.tokens) - s.q0, 0);
  s.k0 = min(max(a.k_starts[b], 0), a.keys);
  s.nk = max(min(a.k_starts[b + 1], a.keys) - s.k0, 0);
  s.shift = s.nk - s.nq;
  return s;
}
// Keys that query i sees: [lo, hi).
TCFP_DEV int key_lo(const Packed& a, const Seq& s, int i) {
  return a.window > 0 ? max(i + s.shift - a.window + 1, 0) : 0;
}
TCFP_DEV int key_hi(const Packed& a, const Seq& s, int i) {
  return a.causal ? min(s.nk, max(i + s.shift + 1, 0)) : s.nk;
}

// Which (sequence, K/V head, member of the group or part, tile) a workgroup
// takes.  Each XCD (workgroup b is on XCD b % 8) has sets of its own, whose K and
// V its L2 then holds; within it the tiles come in order, all sets' first ones
// first.  False: nothing is left for this workgroup.
TCFP_DEV bool place(const Packed& a, int members, int& b, int& kvh, int& member, int& tile) {
  int set, i = int(blockIdx.x);
  if (a.sets >= 8) {
    const int mine = (a.sets + 7) / 8;
    set = i & 7;
    i >>= 3;
    member = i % members;
    i /= members;
    set += 8 * (i % mine);
    tile = i / mine;
  } else {
    member = i % members;
    i /= members;
    set = i % a.sets;
    tile = i / a.sets;
  }
  b = set / a.kv_heads;
  kvh = set - b * a.kv_heads;
  return set < a.sets;
}

// ---- tiles in LDS: kStep rows of D values ------------------------------------
//
// The 16-byte chunks of a row are permuted by swizzle(row), so that reads by rows
// (the same chunk of 16 rows) and transposed ones (64 bytes of four rows) each
// meet every bank once.
template <int D>
TCFP_DEV int swizzle(int row) {
  return D == 64 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
}
template <int D>
constexpr int kTileBytes = kStep * D * 2;

// The wave's share (instructions wave, wave + NW, ...) of the copy of rows
// [row, row + kStep) of x, of which the first `rows` there are.
template <int D, int NW>
TCFP_DEV void copy_tile(const uint16_t* x, int64_t ld, int64_t row, int rows, uint32_t lds,
                        int wave, int lane) {
  constexpr int CH = D / 8, R = 64 / CH, N = kStep / R / NW;
  const v4i rsrc = make_rsrc(
      x + row * ld, rows > 0 ? uint32_t((int64_t(min(rows, kStep) - 1) * ld + D) * 2) : 0u);
  const int r = wave * R + lane / CH;
  const uint32_t off = fresh(r * int(ld) * 2), chunk = fresh(((lane % CH) ^ swizzle<D>(r)) << 4);
  const uint32_t step = uint32_t(NW * R * 2) * uint32_t(ld);
#pragma unroll
  for (int i = 0; i < N; ++i)  // (the swizzle of row i NW R + r is the two's)
    copy16(rsrc, off + (chunk ^ (swizzle<D>(i * NW * R) << 4)) + uint32_t(i) * step,
           lds + uint32_t((i * NW + wave) * 1024));
}

// Where a lane reads its operands of a tile:
// * "rows along lanes": row x + lane % 32, columns 16 d + 8 (lane / 32) ...;
// * "columns along lanes": column 32 x + lane % 32 of the rows r0 + 4 (lane / 32) +
//   {0 ... 3, 8 ... 11}, r0 a multiple of 16: the rows that the lane's accumulators
//   8 (r0 / 16 % 2) ... of a 32-row block hold.
// Both are one offset in which d and x flip bits.
template <int D>
struct Lanes {
  int rows, columns;
  TCFP_DEV void init(int lane) {
    const int row = lane & 31, half = lane >> 5, i = lane & 15, r = 4 * half + (i >> 2);
    rows = row * (2 * D) + ((half ^ swizzle<D>(row)) << 4);
    columns = r * (2 * D) + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ swizzle<D>(r)) << 4) +
              (i & 1) * 8;
  }
};
template <int D>
TCFP_DEV v8bf by_rows(const uint8_t* lds, int off, int x, int d) {
  return read16(lds + (off ^ (d << 5)) + x * (2 * D));
}
template <int D>
TCFP_DEV v8bf by_columns(const uint8_t* lds, int off, int x, int r0) {
  const int at = off ^ (x << 6);
  return read_transposed(lds + at + r0 * (2 * D), lds + (at ^ 32) + (r0 + 8) * (2 * D));
}

// A lane's operand of its own row in memory: columns 16 s + 8 half ....
template <int D>
TCFP_DEV void load_row(const uint16_t* p, int half, bool live, v8bf* f) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (live) w = *reinterpret_cast<const uint4*>(p + 16 * s + 8 * half);
    f[s] = __builtin_bit_cast(v8bf, w);
  }
}
// The sign of the scale, put into one factor of the scores (0: all scores 0).
template <int D>
TCFP_DEV void apply_sign(float sign, v8bf* f) {
  if (sign == 1.0f) return;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    v4i w = __builtin_bit_cast(v4i, f[s]);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = sign == 0.0f ? 0 : w[j] ^ int(0x80008000u);
    f[s] = __builtin_bit_cast(v8bf, w);
  }
}

TCFP_DEV float other_half(float x) { return __shfl_xor(x, 32); }

// Eight accumulators as the bf16 operand of the next product.
TCFP_DEV v8bf pack8(const v16f& e, int z) {
  const v4i w = {int(pack2(e[z], e[z + 1])), int(pack2(e[z + 2], e[z + 3])),
                 int(pack2(e[z + 4], e[z + 5])), int(pack2(e[z + 6], e[z + 7]))};
  return __builtin_bit_cast(v8bf, w);
}
// What that rounding left.
TCFP_DEV v8bf pack8_low(const v16f& e, int z, const v8bf& high) {
  v16f rest;
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = e[z + j] - float(high[j]);
  return pack8(rest, 0);
}
TCFP_DEV v16f zeros() {
  v16f z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.0f;
  return z;
}

// What rounding x to bf16 left, in 2^-8 of bf16's last place: delta = rowsum(dO * O)
// takes O with eight bits more.  From the rounded O alone, short rows lose: dK of
// 32 sequences of 128 tokens was 2.7e-3 off where its own rounding is 1.7e-3.
TCFP_DEV uint32_t low_part(float x) {
  const int bits = __float_as_int(x), high = int(pack2(x, x) & 0xFFFF0000u);
  return uint32_t(min((bits - high + 128) >> 8, 127)) & 0xFFu;
}
TCFP_DEV float with_low(uint32_t high, uint32_t low, int byte) {
  return __int_as_float(int(high) + (int(low << (24 - 8 * byte)) >> 24) * 256);
}

// A wave's transposed result, columns across the registers, as rows of bf16.
template <int D>
TCFP_DEV void store_row(uint16_t* p, const v16f* o, float f, int half) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(p + 32 * i + 8 * g + 4 * half) =
          make_uint2(pack2(o[i][4 * g] * f, o[i][4 * g + 1] * f),
                     pack2(o[i][4 * g + 2] * f, o[i][4 * g + 3] * f));
}

// Rows that belong to no sequence: zeros (by the workgroups of the first and last
// one's first tiles; sequences are one after another, a gap between two is left
// as it is by neither).
template <int D>
TCFP_DEV void zero_rows(uint16_t* x, int from, int to, int heads, int head0, int n) {
  constexpr int CH = D / 8;
  const int64_t items = int64_t(max(to - from, 0)) * n * CH;
  for (int64_t i = threadIdx.x; i < items; i += blockDim.x) {
    const int c = int(i % CH);
    const int64_t rh = i / CH, row = from + rh / n, h = head0 + rh % n;
    *reinterpret_cast<uint4*>(x + (row * heads + h) * D + c * 8) = make_uint4(0, 0, 0, 0);
  }
}

// ---- forward -------------------------------------------------------------------
//
// A workgroup takes 32 NW queries of a head, a wave 32 of them, whose Q stays in
// registers; K and V come in steps of 64 keys, two steps of them in LDS.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void packed_forward_kernel(Packed a) {
  constexpr int TILE = kTileBytes<D>;
  __shared__ __align__(16) uint8_t lds[4 * TILE];  // two steps of K and V
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b, kvh, member, tile;
  if (!place(a, a.group, b, kvh, member, tile)) return;
  const int head = kvh * a.group + member;
  const Seq s = sequence(a, b);
  if (tile == 0) {
    if (b == 0) zero_rows<D>(a.o, 0, s.q0, a.heads, head, 1);
    if (b == a.batch - 1) zero_rows<D>(a.o, s.q0 + s.nq, a.tokens, a.heads, head, 1);
  }
  const uint32_t lds0 = lds_offset(lds);
  Lanes<D> at_lane;
  at_lane.init(lane);
  const int tiles = (s.nq + 32 * NW - 1) / (32 * NW);
  // (the last tiles, which see the most keys, first; a bound on the lengths that
  // is too small gives a workgroup several)
  for (int at = tiles - 1 - tile; at >= 0; at -= a.tiles) {
    const int r0 = at * 32 * NW, last = min(r0 + 32 * NW, s.nq) - 1;
    const int begin = key_lo(a, s, r0) & ~(kStep - 1), end = key_hi(a, s, last);
    const int row = min(r0 + 32 * wave + col, last);
    const int lo = key_lo(a, s, row), hi = key_hi(a, s, row);
    const int wfirst = min(r0 + 32 * wave, last), wlast = min(r0 + 32 * wave + 31, last);
    const int w_lo = key_lo(a, s, wfirst), w_lo_max = key_lo(a, s, wlast),
              w_hi_min = key_hi(a, s, wfirst), w_hi = key_hi(a, s, wlast);
    const bool idle = r0 + 32 * wave > last;
    v8bf q[D / 16];
    load_row<D>(a.q + int64_t(s.q0 + row) * a.q_token + int64_t(head) * a.q_head, half, true, q);
    apply_sign<D>(a.sign, q);
    v16f o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = zeros();
    float m = -INFINITY, l = 0.0f;
    auto fetch = [&](int key, int buf) {
      copy_tile<D, NW>(a.k + int64_t(kvh) * a.k_head, a.k_token, s.k0 + key, s.nk - key,
                       lds0 + uint32_t(buf) * 2 * TILE, wave, lane);
      copy_tile<D, NW>(a.v + int64_t(kvh) * a.v_head, a.v_token, s.k0 + key, s.nk - key,
                       lds0 + uint32_t(buf) * 2 * TILE + TILE, wave, lane);
    };
    if (begin < end) fetch(begin, 0);
    int buf = 0;
    for (int key = begin; key < end; key += kStep, buf ^= 1) {
      wait_and_sync<0>();  // this step is there, the one before it read
      if (key + kStep < end) fetch(key + kStep, buf ^ 1);
      if (idle || key >= w_hi || key + kStep <= w_lo) continue;
      const int k_off = fresh(buf * 2 * TILE + at_lane.rows);
      const int v_off = fresh(buf * 2 * TILE + TILE + at_lane.columns);
      v16f e[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        e[x] = zeros();
#pragma unroll
        for (int d = 0; d < D / 16; ++d) e[x] = mfma(by_rows<D>(lds, k_off, 32 * x, d), q[d], e[x]);
      }
      if (key < w_lo_max || key + kStep > w_hi_min) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = key + 32 * x + 8 * (r >> 2) + 4 * half + (r & 3);
            if (j < lo || j >= hi) e[x][r] = -INFINITY;
          }
      }
      float top = m;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, e[x][r]);
      top = fmaxf(top, other_half(top));
      if (__ballot(top > m)) {
        const float f = top == m ? 1.0f : exp2_fast((m - top) * a.c);
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= f;
      }
      const float off = top == -INFINITY ? 0.0f : top * a.c;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          e[x][r] = exp2_fast(__builtin_fmaf(e[x][r], a.c, -off));
          l += e[x][r];
        }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const v8bf p = pack8(e[x >> 1], 8 * (x & 1));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = mfma(by_columns<D>(lds, v_off, i, 16 * x), p, o[i]);
      }
    }
    l += other_half(l);
    if (r0 + 32 * wave + col <= last) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      // (nothing is seen: a weight of 0 times what others' values hold may be NaN)
      if (l == 0.0f) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = zeros();
      }
      const int64_t at_row = (int64_t(s.q0 + row) * a.heads + head) * D;
      store_row<D>(a.o + at_row, o, inv, half);
      if (a.low) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t w = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) w |= low_part(o[i][4 * g + r] * inv) << (8 * r);
            *reinterpret_cast<uint32_t*>(a.low + at_row + 32 * i + 8 * g + 4 * half) = w;
          }
      }
      if (a.lse && half == 0)
        a.lse[int64_t(head) * a.tokens + s.q0 + row] =
            l == 0.0f ? INFINITY : m * a.c + log2_fast(l);
    }
    __syncthreads();  // (the next tile's copies)
  }
}

// ---- dQ (and delta) --------------------------------------------------------------
//
// As forward, with dO beside Q in registers; a step's two runs of 32 keys one after
// the other.
template <int D, int NW, bool SHORT>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void packed_dq_kernel(Packed a) {
  constexpr int TILE = kTileBytes<D>;
  __shared__ __align__(16) uint8_t lds[4 * TILE];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b, kvh, member, tile;
  if (!place(a, a.group, b, kvh, member, tile)) return;
  const int head = kvh * a.group + member;
  const Seq s = sequence(a, b);
  if (tile == 0) {
    if (b == 0) zero_rows<D>(a.dq, 0, s.q0, a.heads, head, 1);
    if (b == a.batch - 1) zero_rows<D>(a.dq, s.q0 + s.nq, a.tokens, a.heads, head, 1);
  }
  const uint32_t lds0 = lds_offset(lds);
  Lanes<D> at_lane;
  at_lane.init(lane);
  const int tiles = (s.nq + 32 * NW - 1) / (32 * NW);
  for (int at = tiles - 1 - tile; at >= 0; at -= a.tiles) {
    const int r0 = at * 32 * NW, last = min(r0 + 32 * NW, s.nq) - 1;
    const int begin = key_lo(a, s, r0) & ~(kStep - 1), end = key_hi(a, s, last);
    const int row = min(r0 + 32 * wave + col, last);
    const bool live = r0 + 32 * wave + col <= last;
    const int lo = key_lo(a, s, row), hi = key_hi(a, s, row);
    const int wfirst = min(r0 + 32 * wave, last), wlast = min(r0 + 32 * wave + 31, last);
    const int w_lo = key_lo(a, s, wfirst), w_lo_max = key_lo(a, s, wlast),
              w_hi_min = key_hi(a, s, wfirst), w_hi = key_hi(a, s, wlast);
    const bool idle = r0 + 32 * wave > last;
    auto fetch = [&](int key, int buf) {
      copy_tile<D, NW>(a.k + int64_t(kvh) * a.k_head, a.k_token, s.k0 + key, s.nk - key,
                       lds0 + uint32_t(buf) * 2 * TILE, wave, lane);
      copy_tile<D, NW>(a.v + int64_t(kvh) * a.v_head, a.v_token, s.k0 + key, s.nk - key,
                       lds0 + uint32_t(buf) * 2 * TILE + TILE, wave, lane);
    };
    if (begin < end) fetch(begin, 0);
    v8bf q[D / 16], go[D / 16];
    const int64_t hrow = int64_t(s.q0 + row) * a.heads + head;
    load_row<D>(a.q + int64_t(s.q0 + row) * a.q_token + int64_t(head) * a.q_head, half, true, q);
    load_row<D>(a.go + int64_t(s.q0 + row) * a.go_token + int64_t(head) * a.go_head, half, true,
                go);
    float delta = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int64_t at_o = hrow * D + 16 * d + 8 * half;
      const uint4 o = *reinterpret_cast<const uint4*>(a.o + at_o);
      const uint2 low = *reinterpret_cast<const uint2*>(a.low + at_o);
      const uint32_t ow[4] = {o.x, o.y, o.z, o.w}, lw[2] = {low.x, low.y};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t high = j & 1 ? ow[j / 2] & 0xFFFF0000u : ow[j / 2] << 16;
        delta = __builtin_fmaf(with_low(high, lw[j / 4], j % 4), float(go[d][j]), delta);
      }
    }
    delta += other_half(delta);
    const int64_t stat = int64_t(head) * a.tokens + s.q0 + row;
    if (live && half == 0) a.delta[stat] = delta;
    const float lse = a.lse[stat];
    apply_sign<D>(a.sign, q);
    v16f dq[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dq[i] = zeros();
    int buf = 0;
    for (int key = begin; key < end; key += kStep, buf ^= 1) {
      wait_and_sync<0>();
      if (key + kStep < end) fetch(key + kStep, buf ^ 1);
      if (idle || key >= w_hi || key + kStep <= w_lo) continue;
      const bool masked = key < w_lo_max || key + kStep > w_hi_min;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int k_off = fresh(buf * 2 * TILE + at_lane.rows);
        const int kt_off = fresh(buf * 2 * TILE + at_lane.columns);
        v16f e = zeros(), dp = zeros();
#pragma unroll
        for (int d = 0; d < D / 16; ++d) e = mfma(by_rows<D>(lds, k_off, 32 * x, d), q[d], e);
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          dp = mfma(by_rows<D>(lds + TILE, k_off, 32 * x, d), go[d], dp);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          e[r] = exp2_fast(__builtin_fmaf(e[r], a.c, -lse)) * (dp[r] - delta);
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = key + 32 * x + 8 * (r >> 2) + 4 * half + (r & 3);
            if (j < lo || j >= hi) e[r] = 0.0f;
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const v8bf ds = pack8(e, 8 * y);
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            dq[i] = mfma(by_columns<D>(lds, kt_off, i, 32 * x + 16 * y), ds, dq[i]);
          if constexpr (SHORT) {
            const v8bf low = pack8_low(e, 8 * y, ds);
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
              dq[i] = mfma(by_columns<D>(lds, kt_off, i, 32 * x + 16 * y), low, dq[i]);
          }
        }
      }
    }
    if (lse == INFINITY) {  // (nothing is seen, as forward)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) dq[i] = zeros();
    }
    if (live) store_row<D>(a.dq + hrow * D, dq, a.scale, half);
    __syncthreads();
  }
}

// ---- dK and dV ---------------------------------------------------------------------
//
// A workgroup takes 32 NW keys of a K/V head, a wave 32 of them, whose K and V stay
// in registers; the queries of the group's heads (of a part of them, where the keys
// alone would not fill the card) come in steps of 64 with their dO, L and delta.  Of a
// wave's 256 registers 192 hold its K, V, dK and dV (heads of 128): the phases of 32
// queries -- S and dP, P and dS, the sums -- are kept apart, and the other workgroup on
// the CU fills the matrix cores meanwhile.
template <int D, int NW, bool SHORT>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void packed_dkv_kernel(Packed a) {
  constexpr int TILE = kTileBytes<D>, STATS = 2 * kStep * 4, BUF = 2 * TILE + STATS;
  __shared__ __align__(16) uint8_t lds[2 * BUF];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b, kvh, part, tile;
  if (!place(a, a.parts, b, kvh, part, tile)) return;
  const Seq s = sequence(a, b);
  if (tile == 0 && a.parts == 1) {
    for (int w = 0; w < 2; ++w) {
      uint16_t* x = w ? a.dv : a.dk;
      if (b == 0) zero_rows<D>(x, 0, s.k0, a.kv_heads, kvh, 1);
      if (b == a.batch - 1) zero_rows<D>(x, s.k0 + s.nk, a.keys, a.kv_heads, kvh, 1);
    }
  }
  const int heads_each = (a.group + a.parts - 1) / a.parts;
  const int g0 = part * heads_each, g1 = min(g0 + heads_each, a.group);
  const uint32_t lds0 = lds_offset(lds);
  Lanes<D> at_lane;
  at_lane.init(lane);
  for (int j0 = tile * 32 * NW; j0 < s.nk; j0 += a.tiles * 32 * NW) {
    const int last = min(j0 + 32 * NW, s.nk) - 1;
    // queries that see some of the tile's keys
    const int begin = a.causal ? max(j0 - s.shift, 0) & ~(kStep - 1) : 0;
    const int end = a.window > 0 ? min(s.nq, last + a.window - s.shift) : s.nq;
    const int key = min(j0 + 32 * wave + col, last);
    const bool idle = j0 + 32 * wave > last;
    const int wfirst = min(j0 + 32 * wave, last), wlast = min(j0 + 32 * wave + 31, last);
    // the wave's queries: some of its keys are seen in [w_begin, w_end), all of
    // them in [all_begin, all_end)
    const int w_begin = a.causal ? wfirst - s.shift : 0, all_begin = a.causal ? wlast - s.shift : 0;
    const int w_end = a.window > 0 ? wlast + a.window - s.shift : s.nq,
              all_end = min(a.window > 0 ? wfirst + a.window - s.shift : s.nq, s.nq);
    // the lane's key is seen by queries [first, past)
    const int first = a.causal ? key - s.shift : 0;
    const int past = min(a.window > 0 ? key + a.window - s.shift : s.nq, s.nq);
    v8bf k[D / 16], v[D / 16];
    load_row<D>(a.k + int64_t(s.k0 + key) * a.k_token + int64_t(kvh) * a.k_head, half, true, k);
    load_row<D>(a.v + int64_t(s.k0 + key) * a.v_token + int64_t(kvh) * a.v_head, half, true, v);
    apply_sign<D>(a.sign, k);
    v16f dk[D / 32], dv[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dk[i] = zeros(), dv[i] = zeros();
    const int steps = begin < end ? (end - begin + kStep - 1) / kStep : 0;
    const int total = steps * (g1 - g0);
    auto fetch = [&](int g, int at, int buf) {
      const int head = kvh * a.group + g;
      const uint32_t to = lds0 + uint32_t(buf) * BUF;
      copy_tile<D, NW>(a.q + int64_t(head) * a.q_head, a.q_token, s.q0 + at, s.nq - at, to, wave,
                       lane);
      copy_tile<D, NW>(a.go + int64_t(head) * a.go_head, a.go_token, s.q0 + at, s.nq - at,
                       to + TILE, wave, lane);
      // L and delta of the step, one a lane (zeros past the sequence, whose
      // products are masked)
      if (wave < 2) {
        const float* x = (wave ? a.delta : a.lse) + int64_t(head) * a.tokens + s.q0 + at;
        const uint32_t me = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
        copy4(make_rsrc(x, uint32_t(min(s.nq - at, kStep) * 4)), me * 4,
              to + 2 * TILE + uint32_t(wave) * (kStep * 4));
      }
    };
    int g = g0, at = begin, next_g = g0, next_at = begin;
    auto advance = [&]() {
      next_at += kStep;
      if (next_at >= end) next_at = begin, ++next_g;
    };
    if (total > 0) fetch(g, at, 0);
    int buf = 0;
    for (int i = 0; i < total; ++i, buf ^= 1) {
      wait_and_sync<0>();
      g = next_g, at = next_at;
      advance();
      if (i + 1 < total) fetch(next_g, next_at, buf ^ 1);
      const float* stats = reinterpret_cast<const float*>(lds + buf * BUF + 2 * TILE);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r0 = at + 32 * x;
        if (idle || r0 + 32 <= w_begin || r0 >= w_end) continue;
        const int r_off = fresh(buf * BUF + 32 * x * (2 * D) + at_lane.rows);
        const int c_off = fresh(buf * BUF + 32 * x * (2 * D) + at_lane.columns);
        v16f e = zeros(), dp = zeros();
#pragma unroll
        for (int d = 0; d < D / 16; ++d) dp = mfma(by_rows<D>(lds + TILE, r_off, 0, d), v[d], dp);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) e = mfma(by_rows<D>(lds, r_off, 0, d), k[d], e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 l4 = *reinterpret_cast<const float4*>(stats + 32 * x + 8 * g + 4 * half);
          const float4 d4 =
              *reinterpret_cast<const float4*>(stats + kStep + 32 * x + 8 * g + 4 * half);
          const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, de[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = exp2_fast(__builtin_fmaf(e[4 * g + r], a.c, -ls[r]));
            dp[4 * g + r] = p * (dp[4 * g + r] - de[r]);
            e[4 * g + r] = p;
          }
        }
        if (r0 < all_begin || r0 + 32 > all_end) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int qi = r0 + 8 * (r >> 2) + 4 * half + (r & 3);
            if (qi < first || qi >= past) e[r] = 0.0f, dp[r] = 0.0f;
          }
        }
        const v8bf p[2] = {pack8(e, 0), pack8(e, 8)}, ds[2] = {pack8(dp, 0), pack8(dp, 8)};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            dv[j] = mfma(by_columns<D>(lds + TILE, c_off, j, 16 * y), p[y], dv[j]);
            dk[j] = mfma(by_columns<D>(lds, c_off, j, 16 * y), ds[y], dk[j]);
          }
        if constexpr (SHORT) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const v8bf low = pack8_low(dp, 8 * y, ds[y]);
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
              dk[j] = mfma(by_columns<D>(lds, c_off, j, 16 * y), low, dk[j]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (j0 + 32 * wave + col <= last) {
      const int64_t at = int64_t(s.k0 + key) * a.kv_heads + kvh;
      if (a.parts == 1) {
        store_row<D>(a.dk + at * D, dk, a.scale, half);
        store_row<D>(a.dv + at * D, dv, 1.0f, half);
      } else {
        const int64_t whole = int64_t(a.keys) * a.kv_heads * D;
        float* pk = a.part + int64_t(2 * part) * whole + at * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int d = 32 * i + 8 * g + 4 * half;
            *reinterpret_cast<float4*>(pk + d) =
                make_float4(dk[i][4 * g] * a.scale, dk[i][4 * g + 1] * a.scale,
                            dk[i][4 * g + 2] * a.scale, dk[i][4 * g + 3] * a.scale);
            *reinterpret_cast<float4*>(pk + whole + d) =
                make_float4(dv[i][4 * g], dv[i][4 * g + 1], dv[i][4 * g + 2], dv[i][4 * g + 3]);
          }
      }
    }
    __syncthreads();
  }
}

// dK (blockIdx.y 0) and dV (1) from their parts, in order; eight values a thread.
// Rows that belong to no sequence have no parts: zeros.
__global__ __launch_bounds__(256) void packed_join_kernel(Packed a, int64_t eights, int dim) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= eights) return;
  const int64_t whole = eights * 8, row = i * 8 / dim / a.kv_heads;
  const int k_first = min(max(a.k_starts[0], 0), a.keys),
            k_past = min(max(a.k_starts[a.batch], 0), a.keys);
  float v[8] = {};
  if (row >= k_first && row < k_past) {
    const float* p = a.part + int64_t(blockIdx.y) * whole + i * 8;
    for (int s = 0; s < a.parts; ++s, p += 2 * whole) {
      const float4 x = reinterpret_cast<const float4*>(p)[0];
      const float4 y = reinterpret_cast<const float4*>(p)[1];
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
  }
  reinterpret_cast<uint4*>(blockIdx.y ? a.dv : a.dk)[i] =
      make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}

// ---- host ------------------------------------------------------------------------

constexpr int64_t kMostRows = 1 << 29;  // sums of three stay below 2^31
constexpr int kCus = 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int launch_status() { return hipGetLastError() == hipSuccess ? TCFP_OK : TCFP_ERR_HIP; }

// Waves of a workgroup.
constexpr int kWaves = 4;

// Parts of a group's heads in the dK, dV launch, by what they are about to take, us: a
// step of 64 queries, heads of 128, 2.6 for a workgroup alone on a CU and 4.2 beside
// another; the longest chain of steps -- of a causal sequence the first tile of keys has
// twice the mean's -- against all of them over the card; the parts' writing and joining,
// 4.5 TB/s.  (It counts no window and takes every call for causal: tiles whose chains are
// alike are shared out as if they were not, 8192 tokens with 1000 seen back in two parts,
// 539 us the whole backward.)  (32 / 8 heads of 128, the whole backward: one sequence of 8192 4000 us in
// one part, 1770 in two; four of up to 4096 1310 and 1063; six of up to 1000 198 in two,
// 199 in four.)
int parts_of(int64_t keys, int64_t batch, int64_t max_key_len, int kv_heads, int group, int dim) {
  const int64_t rows = 32 * kWaves, longest = std::max<int64_t>(std::min(max_key_len, keys), 1);
  const double tiles =
      double(std::min(ceil_div(longest, rows) * batch, keys / rows + batch) * kv_heads);
  const double steps = double(ceil_div(longest, kStep)) * dim / 128;
  const double slots = dim == 256 ? kCus : 2 * kCus;
  int best = 1;
  double least = INFINITY;
  for (int parts = 1; parts <= group; ++parts) {
    const double step = tiles * parts > kCus ? 4.2 : 2.6;
    const double t = std::max(steps * double(ceil_div(group, parts)) * step,
                              0.5 * steps * group * tiles / slots * 4.2) +
                     (parts > 1 ? 5 + 16 / 4.5e6 * parts * double(keys) * kv_heads * dim : 0);
    if (t < least) least = t, best = parts;
  }
  return best;
}

// (sequence, K/V head)s of a launch: whole rounds of the XCDs, see place().
int64_t sets_of(int64_t batch, int kv_heads) {
  const int64_t sets = batch * kv_heads;
  return sets >= 8 ? (sets + 7) / 8 * 8 : sets;
}

struct Sizes {
  int64_t tokens, keys, batch, max_len, max_key_len, window;
  int heads, kv_heads, dim;
  float scale;
};
int check_sizes(const Sizes& z) {
  if (z.dim != 64 && z.dim != 128 && z.dim != 256) return TCFP_ERR_SHAPE;
  if (z.tokens < 0 || z.keys < 0 || z.tokens > kMostRows || z.keys > kMostRows || z.batch < 0 ||
      z.batch > 65535 || z.heads <= 0 || z.heads > 65535 || z.kv_heads <= 0 ||
      z.heads % z.kv_heads || z.max_len < 0 || z.max_key_len < 0 ||
      z.window < 0 || !std::isfinite(z.scale))
    return TCFP_ERR_SHAPE;
  if ((z.tokens > 0 || z.keys > 0) && z.batch == 0) return TCFP_ERR_SHAPE;
  // (a workgroup for each sequence and head at least: what a grid takes)
  if (!grid_x_fits(sets_of(z.batch, z.kv_heads) * (z.heads / z.kv_heads), 64 * kWaves))
    return TCFP_ERR_SHAPE;
  return TCFP_OK;
}
// Row strides within a descriptor's reach, rows of whole 16-byte vectors.
int check_rows(const void* p, int64_t token, int64_t head) {
  if (!aligned16(p) || token % 8 || head % 8) return TCFP_ERR_ALIGN;
  if (token < 0 || head < 0 || token > (1 << 23)) return TCFP_ERR_SHAPE;
  return TCFP_OK;
}
Packed arguments(const Sizes& z, bool causal) {
  Packed a{};
  a.batch = int(z.batch);
  a.tokens = int(z.tokens);
  a.keys = int(z.keys);
  a.heads = z.heads;
  a.kv_heads = z.kv_heads;
  a.group = z.heads / z.kv_heads;
  a.scale = z.scale;
  a.c = z.scale == 0.0f ? 1.0f : std::abs(z.scale) * kLog2e;
  a.sign = z.scale == 0.0f ? 0.0f : z.scale < 0.0f ? -1.0f : 1.0f;
  a.causal = causal;
  a.window = int(std::min<int64_t>(z.window, kMostRows));
  a.sets = int(z.batch * z.kv_heads);
  return a;
}
// Tiles of a sequence and head in a launch with `members` of each set, and its workgroups.
// A bound far past the lengths (all keys of a batch of many sequences) is cut: a
// workgroup takes the tiles that are left over, one after another.  So a launch holds 4
// million workgroups at most, or one for each set and member where those are more.
int64_t lay_out(Packed& a, int64_t max_len, int64_t rows, int members) {
  const int64_t each = sets_of(a.batch, a.kv_heads) * members;
  const int64_t most = std::max<int64_t>((int64_t(1) << 22) / each, 1);
  a.tiles = int(std::clamp<int64_t>(ceil_div(std::min(max_len, rows), 32 * kWaves), 1, most));
  return each * a.tiles;
}

#define TCFP_PACKED(GRID, KERNEL, ...)                                                      \
  do {                                                                                      \
    const int64_t n_ = GRID;                                                                \
    if (n_ > INT32_MAX || !grid_x_fits(n_, 64 * kWaves)) return TCFP_ERR_SHAPE;             \
    const unsigned g_ = unsigned(n_), t_ = 64 * kWaves;                                     \
    if (z.dim == 64) KERNEL<64, kWaves __VA_ARGS__><<<g_, t_, 0, st>>>(a);                  \
    else if (z.dim == 128) KERNEL<128, kWaves __VA_ARGS__><<<g_, t_, 0, st>>>(a);           \
    else KERNEL<256, kWaves __VA_ARGS__><<<g_, t_, 0, st>>>(a);                             \
    if (launch_status() != TCFP_OK) return TCFP_ERR_HIP;                                    \
  } while (0)

}  // namespace

extern "C" {

int tcfp_packed_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                          const void* k, int64_t k_token_stride, int64_t k_head_stride,
                          const void* v, int64_t v_token_stride, int64_t v_head_stride,
                          const int32_t* q_starts, const int32_t* k_starts, int64_t batch,
                          int64_t tokens, int64_t keys, int heads, int kv_heads, int dim,
                          int64_t max_len, float scale, int causal, int64_t window, void* out,
                          int8_t* out_low, float* lse, void* stream) {
  const Sizes z{tokens, keys, batch, max_len, 0, window, heads, kv_heads, dim, scale};
  if (const int rc = check_sizes(z)) return rc;
  if (const int rc = check_rows(q, q_token_stride, q_head_stride)) return rc;
  if (const int rc = check_rows(k, k_token_stride, k_head_stride)) return rc;
  if (const int rc = check_rows(v, v_token_stride, v_head_stride)) return rc;
  if (!aligned16(out) || !aligned16(out_low)) return TCFP_ERR_ALIGN;
  if (tokens == 0) return TCFP_OK;
  Packed a = arguments(z, causal != 0);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_token = q_token_stride; a.q_head = q_head_stride;
  a.k_token = k_token_stride; a.k_head = k_head_stride;
  a.v_token = v_token_stride; a.v_head = v_head_stride;
  a.q_starts = q_starts;
  a.k_starts = k_starts;
  a.o = static_cast<uint16_t*>(out);
  a.low = out_low;
  a.lse = lse;
  const auto st = static_cast<hipStream_t>(stream);
  TCFP_PACKED(lay_out(a, max_len, tokens, a.group), packed_forward_kernel);
  return TCFP_OK;
}

size_t tcfp_packed_attention_backward_workspace_bytes(int64_t tokens, int64_t keys, int64_t batch,
                                                      int64_t max_key_len, int heads, int kv_heads,
                                                      int dim) {
  if (tokens < 0 || keys < 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return 0;
  const int parts = parts_of(keys, batch, max_key_len, kv_heads, heads / kv_heads, dim);
  return align256(size_t(tokens) * size_t(heads) * 4) +
         (parts > 1 ? size_t(parts) * 2 * size_t(keys) * size_t(kv_heads) * size_t(dim) * 4 : 0);
}

int tcfp_packed_attention_backward(
    const void* grad_out, int64_t go_token_stride, int64_t go_head_stride, const void* q,
    int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
    int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
    const void* out, const int8_t* out_low, const float* lse, const int32_t* q_starts,
    const int32_t* k_starts, int64_t batch, int64_t tokens, int64_t keys, int heads, int kv_heads,
    int dim, int64_t max_len, int64_t max_key_len, float scale, int causal, int64_t window,
    void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, keys, batch, max_len, max_key_len, window, heads, kv_heads, dim, scale};
  if (const int rc = check_sizes(z)) return rc;
  if (const int rc = check_rows(grad_out, go_token_stride, go_head_stride)) return rc;
  if (const int rc = check_rows(q, q_token_stride, q_head_stride)) return rc;
  if (const int rc = check_rows(k, k_token_stride, k_head_stride)) return rc;
  if (const int rc = check_rows(v, v_token_stride, v_head_stride)) return rc;
  if (!aligned16(out) || !aligned16(out_low) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return TCFP_ERR_ALIGN;
  if (tokens == 0 && keys == 0) return TCFP_OK;
  const size_t need = tcfp_packed_attention_backward_workspace_bytes(
      tokens, keys, batch, max_key_len, heads, kv_heads, dim);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return TCFP_ERR_WORKSPACE;
  Packed a = arguments(z, causal != 0);
  a.go = static_cast<const uint16_t*>(grad_out);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.go_token = go_token_stride; a.go_head = go_head_stride;
  a.q_token = q_token_stride; a.q_head = q_head_stride;
  a.k_token = k_token_stride; a.k_head = k_head_stride;
  a.v_token = v_token_stride; a.v_head = v_head_stride;
  a.q_starts = q_starts;
  a.k_starts = k_starts;
  a.o = const_cast<uint16_t*>(static_cast<const uint16_t*>(out));
  a.low = const_cast<int8_t*>(out_low);
  a.lse = const_cast<float*>(lse);
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.delta = static_cast<float*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                    align256(size_t(tokens) * size_t(heads) * 4));
  const auto st = static_cast<hipStream_t>(stream);
  const bool brief = std::max(max_len, max_key_len) <= kShort;
  if (tokens > 0) {
    const int64_t grid = lay_out(a, max_len, tokens, a.group);
    if (brief) TCFP_PACKED(grid, packed_dq_kernel, , true);
    else TCFP_PACKED(grid, packed_dq_kernel, , false);
  }
  if (keys > 0) {
    a.parts = parts_of(keys, batch, max_key_len, kv_heads, a.group, dim);
    const int64_t grid = lay_out(a, max_key_len, keys, a.parts);
    if (brief) TCFP_PACKED(grid, packed_dkv_kernel, , true);
    else TCFP_PACKED(grid, packed_dkv_kernel, , false);
    if (a.parts > 1) {
      const int64_t eights = keys * kv_heads * dim / 8, blocks = ceil_div(eights, 256);
      if (!grid_x_fits(blocks, 256)) return TCFP_ERR_SHAPE;
      packed_join_kernel<<<dim3(unsigned(blocks), 2), 256, 0, st>>>(a, eights, dim);
      return launch_status();
    }
  }
  return TCFP_OK;
}

}  // extern "C"
