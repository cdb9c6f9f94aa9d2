// Residual addition + root-mean-square norm, with an output in FP8 codes and
// block scales or in plain values, and its backward, for gfx950.
//
//   s = x + r,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s * rstd * w
//   dx = rstd * (g - xh * mean(g * xh)) + gh,  g = gy * w,  xh = h * rstd
//   dw = sum over rows of gy * xh
#include <algorithm>

#include "common.h"

using namespace tcfp;

namespace {

constexpr int kThreads = 256;

inline int launch_status() { return hipGetLastError() == hipSuccess ? TCFP_OK : TCFP_ERR_HIP; }
inline bool dtype_ok(int t) { return t == TCFP_DTYPE_F32 || t == TCFP_DTYPE_BF16; }

TCFP_DEV float load1(const void* p, int dtype, int64_t i) {
  return dtype == TCFP_DTYPE_BF16 ? bf16_to_f32(static_cast<const uint16_t*>(p)[i])
                                  : static_cast<const float*>(p)[i];
}
TCFP_DEV void store1(void* p, int dtype, int64_t i, float v) {
  if (dtype == TCFP_DTYPE_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16_rne(v);
  else static_cast<float*>(p)[i] = v;
}

TCFP_DEV float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Sum over the workgroup's waves in wave order, to every thread; `red` holds a
// float per wave and is free again after the caller's next barrier.
template <int T>
TCFP_DEV float block_sum(float v, float* red) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) v += red[i];
  return v;
}

// to_fp8's scale rule on an fp32 block: 448 * (1 / amax) and its inverse.
TCFP_DEV void scale_of(float amax, float fmax, float& mul, float& inv) {
  const float a = amax != amax ? amax : fmaxf(amax, 1e-12f);
  mul = __fmul_rn(__fdiv_rn(1.0f, a), fmax);
  inv = __fdiv_rn(1.0f, mul);
}

struct Norm {
  const void* x;
  const void* r;
  const void* w;
  int64_t ldx, ldr;
  int x_dtype, r_dtype, w_dtype, y_dtype;
  int64_t rows;
  int64_t cols;
  float eps;
  int block, fmt, f32_scales;
  void* h;
  void* y;
  uint8_t* q;
  void* scales;
  float* rstd;
};

// One workgroup a row, any width and alignment: the row is read twice, the
// second time from L2.  Blocks of the quantised output are groups of 32
// consecutive threads, an element each, stepping over a block's columns.
template <bool QUANT>
__global__ __launch_bounds__(kThreads) void norm_any_kernel(Norm a) {
  __shared__ float red[kThreads / 64];
  const int64_t row = blockIdx.x;
  auto sum_at = [&](int64_t c) {
    float s = load1(a.x, a.x_dtype, row * a.ldx + c);
    if (a.r) s += load1(a.r, a.r_dtype, row * a.ldr + c);
    return s;
  };
  float ss = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
    const float s = sum_at(c);
    if (a.h) store1(a.h, a.r_dtype, row * a.cols + c, s);
    ss += s * s;
  }
  ss = block_sum<kThreads>(ss, red);
  const float rstd = 1.0f / sqrtf(ss / float(a.cols) + a.eps);
  if (threadIdx.x == 0) a.rstd[row] = rstd;
  if constexpr (!QUANT) {
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads)
      store1(a.y, a.y_dtype, row * a.cols + c, sum_at(c) * rstd * load1(a.w, a.w_dtype, c));
  } else {
    const int lane = threadIdx.x & 31;
    const float fmax = fp8_max(a.fmt);
    for (int64_t kb = threadIdx.x >> 5; kb < a.cols / a.block; kb += kThreads / 32) {
      uint32_t m = 0;
      for (int j = lane; j < a.block; j += 32) {
        const int64_t c = kb * a.block + j;
        m = umax(m, absbits(sum_at(c) * rstd * load1(a.w, a.w_dtype, c)));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = umax(m, uint32_t(__shfl_xor(int(m), o, 32)));
      float mul, inv = 0.0f;
      int e = 0;
      if (a.f32_scales) {
        scale_of(__uint_as_float(m), fmax, mul, inv);
      } else {
        e = block_exponent(__uint_as_float(m), fmax);
        mul = exp2i(-e);
      }
      for (int j = lane; j < a.block; j += 32) {
        const int64_t c = kb * a.block + j;
        const float v = clampf(sum_at(c) * rstd * load1(a.w, a.w_dtype, c) * mul, fmax);
        a.q[row * a.cols + c] =
            uint8_t(a.fmt == TCFP_FP8_E5M2 ? f32_to_e5m2(v) : f32_to_e4m3(v));
      }
      if (lane == 0) {
        if (a.f32_scales) static_cast<float*>(a.scales)[kb * a.rows + row] = inv;
        else static_cast<int8_t*>(a.scales)[kb * a.rows + row] = int8_t(e);
      }
    }
  }
}

// ---- rows held in registers --------------------------------------------------
//
// Bound by HBM: each input is read and each output written once.  T threads
// hold a row, C vectors of 8 neighbouring elements each (vector i of thread t
// at column 8 (t + i T)), so a block's maximum is over 4, 8 or 16 neighbouring
// lanes.  One row for each T threads of the launch: thousands of small
// workgroups keep more loads in flight than few that walk rows with the next
// row prefetched (8192 x 4096 bf16 + residual: 47.6 us against 51 / 60 / 63 at
// 2 / 8 / 16 rows a workgroup).  Now 47.0 us there (5.0 TB/s), 161 us at 65536 x
// 2048 (5.8 TB/s), 2.8 us for a single row of 4096 (a launch and two latencies).
// (NT: with the non-temporal hint)
template <bool NT>
TCFP_DEV uint4 load16(const void* p) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u* q = static_cast<const v4u*>(p);
  const v4u t = NT ? __builtin_nontemporal_load(q) : *q;
  return make_uint4(t.x, t.y, t.z, t.w);
}
template <typename T>
struct Raw8;
template <>
struct Raw8<uint16_t> {
  uint4 a;
  template <bool NT = false>
  TCFP_DEV void load(const uint16_t* p) {
    a = load16<NT>(p);
  }
  TCFP_DEV void zero() { a = make_uint4(0, 0, 0, 0); }
  TCFP_DEV void get(float* v) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  template <bool NT = false>
  TCFP_DEV void load(const float* p) {
    a = __builtin_bit_cast(float4, load16<NT>(p));
    b = __builtin_bit_cast(float4, load16<NT>(p + 4));
  }
  TCFP_DEV void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  TCFP_DEV void get(float* v) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};
TCFP_DEV uint32_t pack_bf16(float a, float b) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, r);
}
template <bool NT>
TCFP_DEV void store16(void* p, uint4 v) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u t = {v.x, v.y, v.z, v.w};
  if constexpr (NT) __builtin_nontemporal_store(t, static_cast<v4u*>(p));
  else *static_cast<v4u*>(p) = t;
}
template <bool NT = false>
TCFP_DEV void store8(uint16_t* p, const float* v) {
  store16<NT>(p, make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                            pack_bf16(v[6], v[7])));
}
template <bool NT = false>
TCFP_DEV void store8(float* p, const float* v) {
  store16<NT>(p, __builtin_bit_cast(uint4, make_float4(v[0], v[1], v[2], v[3])));
  store16<NT>(p + 4, __builtin_bit_cast(uint4, make_float4(v[4], v[5], v[6], v[7])));
}
TCFP_DEV void load8_any(const void* p, int dtype, int64_t i, float* v) {
  if (dtype == TCFP_DTYPE_BF16) {
    Raw8<uint16_t> r;
    r.load(static_cast<const uint16_t*>(p) + i);
    r.get(v);
  } else {
    Raw8<float> r;
    r.load(static_cast<const float*>(p) + i);
    r.get(v);
  }
}

// Threads of a workgroup whose rows take T of them.
constexpr int wg_of(int t) { return t > kThreads ? t : kThreads; }

// Sum over the T threads of a row, to each of them, through `red` (a float per
// wave of the workgroup) where a row is more than a wave.
template <int T>
TCFP_DEV float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (T > 64) {
    const int first = threadIdx.x / T * (T / 64);
    red[threadIdx.x >> 6] = v;  // (every lane of the wave the same)
    __syncthreads();
    v = red[first];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) v += red[first + i];
  }
  return v;
}

template <typename XT, typename RT, bool QUANT, bool NT, int T, int C>
__global__ __launch_bounds__(wg_of(T)) void norm_rows_kernel(Norm a) {
  constexpr int G = wg_of(T) / T;  // rows of a workgroup
  __shared__ float red[wg_of(T) / 64];
  __shared__ uint32_t sc[QUANT ? G * T * C / 4 : 1];  // scales of its blocks of 32 columns or more
  const int t = threadIdx.x % T, g = threadIdx.x / T;
  const int64_t row = int64_t(blockIdx.x) * G + g;
  const bool live = row < a.rows;
  const int nvec = int(a.cols / 8);
  const XT* x = static_cast<const XT*>(a.x);
  const RT* r = static_cast<const RT*>(a.r);
  Raw8<XT> nx[C];
  Raw8<RT> nr[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int v = t + i * T;
    nx[i].zero();
    nr[i].zero();
    if (v < nvec && live) {
      nx[i].template load<NT>(x + row * a.ldx + v * 8);
      if (r) nr[i].template load<NT>(r + row * a.ldr + v * 8);
    }
  }
  float w[C][8] = {};
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (t + i * T < nvec) load8_any(a.w, a.w_dtype, (t + i * T) * 8, w[i]);
  float s[C][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    nx[i].get(s[i]);
    if (r) {
      float rv[8];
      nr[i].get(rv);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] += rv[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(s[i][j], s[i][j], ss);
  }
  if (a.h && live) {
    // (not read again before the layer between is done: non-temporal, which
    // leaves the L2 to the rest: 48.5 us against 50.8 at 8192 x 4096, 7.9
    // against 9.0 at 4096 x 1024)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (t + i * T < nvec)
        store8<true>(static_cast<RT*>(a.h) + row * a.cols + (t + i * T) * 8, s[i]);
  }
  ss = row_sum<T>(ss, red);
  const float rstd = 1.0f / sqrtf(ss / float(a.cols) + a.eps);
  if (t == 0 && live) a.rstd[row] = rstd;
  const float fmax = fp8_max(a.fmt);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int v = t + i * T;
    const bool mine = live && v < nvec;
    const int64_t at = row * a.cols + v * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[i][j] = s[i][j] * rstd * w[i][j];
    if constexpr (!QUANT) {
      if (!mine) continue;
      if (a.y_dtype == TCFP_DTYPE_BF16) store8(static_cast<uint16_t*>(a.y) + at, s[i]);
      else store8(static_cast<float*>(a.y) + at, s[i]);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = umax(m, absbits(s[i][j]));
      if (a.block == 32) m = seg_umax<4>(m);
      else if (a.block == 64) m = seg_umax<8>(m);
      else m = seg_umax<16>(m);
      float mul, inv = 0.0f;
      int e = 0;
      if (a.f32_scales) {
        scale_of(__uint_as_float(m), fmax, mul, inv);
      } else {
        e = block_exponent(__uint_as_float(m), fmax);
        mul = exp2i(-e);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = clampf(s[i][j] * mul, fmax);
      uint2 q;
      if (a.fmt == TCFP_FP8_E5M2)
        q = make_uint2(cvt4_fp8<TCFP_FP8_E5M2>(s[i][0], s[i][1], s[i][2], s[i][3]),
                       cvt4_fp8<TCFP_FP8_E5M2>(s[i][4], s[i][5], s[i][6], s[i][7]));
      else
        q = make_uint2(cvt4_fp8<TCFP_FP8_E4M3>(s[i][0], s[i][1], s[i][2], s[i][3]),
                       cvt4_fp8<TCFP_FP8_E4M3>(s[i][4], s[i][5], s[i][6], s[i][7]));
      if (!mine) continue;
      *reinterpret_cast<uint2*>(a.q + at) = q;
      if ((v * 8) % a.block == 0)
        sc[v * 8 / a.block * G + g] = a.f32_scales ? __float_as_uint(inv) : uint32_t(e);
    }
  }
  if constexpr (QUANT) {
    // the scales, gathered, so that whole waves write them
    __syncthreads();
    const int64_t row0 = int64_t(blockIdx.x) * G;
    for (int i = threadIdx.x; i < int(a.cols / a.block) * G; i += wg_of(T)) {
      if (row0 + i % G >= a.rows) continue;
      const int64_t at = int64_t(i / G) * a.rows + row0 + i % G;
      if (a.f32_scales) static_cast<uint32_t*>(a.scales)[at] = sc[i];
      else static_cast<int8_t*>(a.scales)[at] = int8_t(sc[i]);
    }
  }
}

// Threads and vectors of a row: two vectors a thread where the rows fill the
// card, one where there are few (latency); t == 0: the kernel for any row.
constexpr int64_t kManyRows = 1024;
struct RowShape {
  int t, c;
};
RowShape row_shape(int64_t rows, int64_t cols) {
  if (cols % 8 != 0 || cols > 1024 * 16) return {0, 0};
  const int64_t nvec = cols / 8;
  int t = 64;
  if (rows >= kManyRows) {
    while (t * 2 < nvec) t *= 2;
  } else {
    while (t < nvec && t < 1024) t *= 2;
  }
  return {t, t < nvec ? 2 : 1};
}
bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t size_of(int dtype) { return dtype == TCFP_DTYPE_BF16 ? 2 : 4; }

// Inputs of more than 96 MiB, three eighths of the cache behind the L2s, are read
// with the non-temporal hint (8192 x 4096 bf16 + residual, 128 MiB: forward 50.0 us
// against 52.9; backward, 192 MiB, 52.4 against 57.0); smaller ones, which their
// producer may have left there, are not (8192 x 1024: 13.3 us against 14.8 with it,
// 16.7 against 18.6).
constexpr int64_t kStreamBytes = 96ll << 20;

#define TCFP_ROWS(CALL)                              \
  do {                                               \
    const bool one = s.c == 1;                       \
    if (s.t == 64 && one) CALL(64, 1);               \
    else if (s.t == 64) CALL(64, 2);                 \
    else if (s.t == 128 && one) CALL(128, 1);        \
    else if (s.t == 128) CALL(128, 2);               \
    else if (s.t == 256 && one) CALL(256, 1);        \
    else if (s.t == 256) CALL(256, 2);               \
    else if (s.t == 512 && one) CALL(512, 1);        \
    else if (s.t == 512) CALL(512, 2);               \
    else if (one) CALL(1024, 1);                     \
    else CALL(1024, 2);                              \
  } while (0)

// Those that inputs past kStreamBytes come in: a vector a thread only where rows
// are short (with fewer than kManyRows rows, 8192 wide at most, 12 bytes a column at
// most, none is that large).
static_assert((kManyRows - 1) * 8192 * 12 <= kStreamBytes, "no one-vector form is streamed");
#define TCFP_ROWS_STREAM(CALL, WIDEST)               \
  do {                                               \
    if (s.t == 64 && s.c == 1) CALL(64, 1);          \
    else if (s.t == 64) CALL(64, 2);                 \
    else if (s.t == 128) CALL(128, 2);               \
    else if (s.t == 256) CALL(256, 2);               \
    else if (s.t == 512 && s.c == 2) CALL(512, 2);   \
    else WIDEST;                                     \
  } while (0)

template <typename XT, typename RT, bool QUANT>
int norm_rows_launch(const Norm& a, RowShape s, hipStream_t st) {
  const int g = wg_of(s.t) / s.t;
  const unsigned blocks = unsigned((a.rows + g - 1) / g);
  if (!grid_x_fits(blocks, wg_of(s.t))) return TCFP_ERR_SHAPE;
  const int64_t in = a.rows * a.cols * (size_of(a.x_dtype) + (a.r ? size_of(a.r_dtype) : 0));
#define TCFP_NR(T, C) norm_rows_kernel<XT, RT, QUANT, false, T, C><<<blocks, wg_of(T), 0, st>>>(a)
#define TCFP_NR_NT(T, C) norm_rows_kernel<XT, RT, QUANT, true, T, C><<<blocks, wg_of(T), 0, st>>>(a)
  if (in > kStreamBytes) TCFP_ROWS_STREAM(TCFP_NR_NT, TCFP_NR_NT(1024, 2));
  else TCFP_ROWS(TCFP_NR);
#undef TCFP_NR_NT
#undef TCFP_NR
  return launch_status();
}

struct NormBack {
  const void* gy;
  const void* h;
  const float* rstd;
  const void* w;
  const void* gh;
  int gy_dtype, h_dtype, w_dtype;
  int64_t rows, cols;
  void* dx;
  float* part;
};

__global__ __launch_bounds__(kThreads) void norm_dx_any_kernel(NormBack a) {
  __shared__ float red[kThreads / 64];
  const int64_t row = blockIdx.x;
  const float rstd = a.rstd[row];
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
    const int64_t i = row * a.cols + c;
    s += load1(a.gy, a.gy_dtype, i) * load1(a.w, a.w_dtype, c) * (load1(a.h, a.h_dtype, i) * rstd);
  }
  const float mean = block_sum<kThreads>(s, red) / float(a.cols);
  for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
    const int64_t i = row * a.cols + c;
    const float g = load1(a.gy, a.gy_dtype, i) * load1(a.w, a.w_dtype, c);
    float d = rstd * (g - load1(a.h, a.h_dtype, i) * rstd * mean);
    if (a.gh) d += load1(a.gh, a.h_dtype, i);
    store1(a.dx, a.h_dtype, i, d);
  }
}

// Partial column sums of gy * xh over a workgroup's run of rows.
__global__ __launch_bounds__(kThreads) void norm_dw_any_kernel(NormBack a, int64_t per) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t lo = int64_t(blockIdx.y) * per, hi = min(lo + per, a.rows);
  if (c >= a.cols) return;
  float s = 0.0f;
  for (int64_t r = lo; r < hi; ++r) {
    const int64_t i = r * a.cols + c;
    s += load1(a.gy, a.gy_dtype, i) * (load1(a.h, a.h_dtype, i) * a.rstd[r]);
  }
  a.part[int64_t(blockIdx.y) * a.cols + c] = s;
}

// ---- the backward with rows in registers -------------------------------------
//
// Bound by HBM like the forward (8192 x 4096 bf16 with the residual's gradient:
// 53 us with the joining launch, 5.1 TB/s; 65536 x 2048 5.8 TB/s), at a thousand
// rows by latency (1000 x 1056 fp32 9.1 us: two dependent launches of 5.5 and 3.4).
// Workgroups take every gridDim.x-th group of rows, the next rows' loads in
// flight; a thread's columns are the same in all its rows, so it sums its share
// of dw in registers, the workgroup leaves one partial row and a second launch
// adds the partials, in an order that the sizes fix.
template <typename GT, typename HT, bool NT, int T, int C>
__global__ __launch_bounds__(wg_of(T)) void norm_back_rows_kernel(NormBack a) {
  constexpr int G = wg_of(T) / T;
  __shared__ float red[2][wg_of(T) / 64];
  __shared__ float4 dws[G > 1 ? (G - 1) * T * C * 2 : 1];
  const int t = threadIdx.x % T, g = threadIdx.x / T;
  const int nvec = int(a.cols / 8);
  const GT* gy = static_cast<const GT*>(a.gy);
  const HT* h = static_cast<const HT*>(a.h);
  const HT* gh = static_cast<const HT*>(a.gh);
  float w[C][8], dw[C][8];
  Raw8<GT> ng[C];
  Raw8<HT> nh[C], na[C];
  float nrs = 0.0f;
  auto fetch = [&](int64_t row) {
    const bool live = row < a.rows;
    nrs = live ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = t + i * T;
      if (v < nvec && live) {
        const int64_t at = row * a.cols + v * 8;
        ng[i].template load<NT>(gy + at);
        nh[i].template load<NT>(h + at);
        if (gh) na[i].template load<NT>(gh + at);
      } else {
        ng[i].zero();
        nh[i].zero();
        na[i].zero();
      }
    }
  };
  fetch(int64_t(blockIdx.x) * G + g);
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[i][j] = dw[i][j] = 0.0f;
    if (t + i * T < nvec) load8_any(a.w, a.w_dtype, (t + i * T) * 8, w[i]);
  }
  const float inv_n = 1.0f / float(a.cols);
  int parity = 0;
  for (int64_t row0 = int64_t(blockIdx.x) * G; row0 < a.rows; row0 += int64_t(gridDim.x) * G) {
    const int64_t row = row0 + g;
    const float rs = nrs;
    float gg[C][8], xh[C][8], add[C][8];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      ng[i].get(gg[i]);
      nh[i].get(xh[i]);
      if (gh) na[i].get(add[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] *= rs;
        dw[i][j] = __builtin_fmaf(gg[i][j], xh[i][j], dw[i][j]);
        gg[i][j] *= w[i][j];
        s = __builtin_fmaf(gg[i][j], xh[i][j], s);
      }
    }
    fetch(row + int64_t(gridDim.x) * G);
    s = row_sum<T>(s, red[parity]) * inv_n;  // (one barrier a row: two arrays in turn)
    parity ^= 1;
    if (row < a.rows) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int v = t + i * T;
        if (v >= nvec) continue;
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d[j] = rs * (gg[i][j] - xh[i][j] * s);
          if (gh) d[j] += add[i][j];
        }
        store8(static_cast<HT*>(a.dx) + row * a.cols + v * 8, d);
      }
    }
  }
  if (!a.part) return;
  if constexpr (G > 1) {
    if (g > 0) {
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          dws[(((g - 1) * C + i) * 2 + j) * T + t] =
              make_float4(dw[i][4 * j], dw[i][4 * j + 1], dw[i][4 * j + 2], dw[i][4 * j + 3]);
    }
    __syncthreads();
    if (g > 0) return;
    for (int x = 0; x < G - 1; ++x)
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 o = dws[((x * C + i) * 2 + j) * T + t];
          dw[i][4 * j] += o.x; dw[i][4 * j + 1] += o.y;
          dw[i][4 * j + 2] += o.z; dw[i][4 * j + 3] += o.w;
        }
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (t + i * T < nvec)
      store8(a.part + int64_t(blockIdx.x) * a.cols + (t + i * T) * 8, dw[i]);
}

// The backward holds three inputs, dw and w of a row: two vectors for each of
// 1024 threads would spill.
RowShape back_shape(int64_t rows, int64_t cols) {
  const RowShape s = row_shape(rows, cols);
  return s.t == 1024 && s.c == 2 ? RowShape{512, 4} : s;
}

template <typename GT, typename HT, bool NT>
void norm_back_launch(const NormBack& a, RowShape s, unsigned blocks, hipStream_t st) {
#define TCFP_NB(T, C) norm_back_rows_kernel<GT, HT, NT, T, C><<<blocks, wg_of(T), 0, st>>>(a)
#define TCFP_NB_SMALL(T, C) TCFP_NB(T, (T) == 1024 ? 1 : (C))
  if constexpr (NT) TCFP_ROWS_STREAM(TCFP_NB, TCFP_NB(512, 4));
  else if (s.c == 4) TCFP_NB(512, 4);
  else TCFP_ROWS(TCFP_NB_SMALL);
#undef TCFP_NB_SMALL
#undef TCFP_NB
}

// dw from the partial rows: a workgroup 16 columns, its threads 64 partials at a
// time (a few loads in a row each: what is left is latency), then the lanes' and
// the waves' sums in order.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void norm_dw_sum_kernel(const float* part, int parts,
                                                                  int64_t cols, float* dw) {
  __shared__ float s[kSumThreads / 64][16];
  const int c = threadIdx.x & 15, p0 = threadIdx.x >> 4;
  const int64_t col = int64_t(blockIdx.x) * 16 + c;
  float v = 0.0f;
  if (col < cols) {
#pragma unroll 4
    for (int p = p0; p < parts; p += kSumThreads / 16) v += part[int64_t(p) * cols + col];
  }
  v += __shfl_xor(v, 16, 64);
  v += __shfl_xor(v, 32, 64);
  if ((threadIdx.x & 63) < 16) s[threadIdx.x >> 6][c] = v;
  __syncthreads();
  if (threadIdx.x < 16 && col < cols) {
#pragma unroll
    for (int i = 1; i < kSumThreads / 64; ++i) v += s[i][c];
    dw[col] = v;
  }
}

// Workgroups of the backward, each a partial row of dw: as many as a CU holds
// of them at a time (three of 256 threads, one of 512 or 1024; a part of a
// second round costs as much as a whole one: 8192 x 8192 bf16 115 us with 256,
// 140 with 384), fewer where there are few rows, at least two each.
int64_t parts_of(int64_t rows, int64_t cols) {
  const RowShape s = back_shape(rows, cols);
  return std::clamp<int64_t>(rows / 2, 1, s.t > 256 ? 256 : rows <= 4096 ? 512 : 768);
}

int norm_checks(const Norm& a, bool quantised) {
  if (a.rows < 0 || a.cols < 0 || a.rows > INT32_MAX || a.cols > INT32_MAX) return TCFP_ERR_SHAPE;
  if (a.ldx < a.cols || (a.r && a.ldr < a.cols)) return TCFP_ERR_SHAPE;
  if (!dtype_ok(a.x_dtype) || !dtype_ok(a.w_dtype) || (a.r && !dtype_ok(a.r_dtype)))
    return TCFP_ERR_DTYPE;
  if (a.h && !a.r) return TCFP_ERR_SHAPE;
  if (quantised) {
    if (a.block != 32 && a.block != 64 && a.block != 128) return TCFP_ERR_SHAPE;
    if (a.cols % a.block != 0) return TCFP_ERR_SHAPE;
    if (a.fmt != TCFP_FP8_E4M3 && a.fmt != TCFP_FP8_E5M2) return TCFP_ERR_DTYPE;
    if (reinterpret_cast<uintptr_t>(a.q) & 7u) return TCFP_ERR_ALIGN;
  } else if (!dtype_ok(a.y_dtype)) {
    return TCFP_ERR_DTYPE;
  }
  return TCFP_OK;
}

template <bool QUANT>
int norm_launch(const Norm& a, hipStream_t st) {
  const int rc = norm_checks(a, QUANT);
  if (rc != TCFP_OK || a.rows == 0) return rc;  // (rows without columns have their rstd, NaN)
  const RowShape s = row_shape(a.rows, a.cols);
  const int64_t xs = size_of(a.x_dtype), rs = size_of(a.r_dtype);
  const bool vec = aligned(a.x, 16) && a.ldx * xs % 16 == 0 && aligned(a.w, 16) &&
                   (!a.r || (aligned(a.r, 16) && a.ldr * rs % 16 == 0)) && aligned(a.h, 16) &&
                   aligned(a.y, 16);
  if (s.t && vec) {
    const bool xb = a.x_dtype == TCFP_DTYPE_BF16;
    const bool rb = a.r ? a.r_dtype == TCFP_DTYPE_BF16 : xb;
    if (xb) return rb ? norm_rows_launch<uint16_t, uint16_t, QUANT>(a, s, st)
                      : norm_rows_launch<uint16_t, float, QUANT>(a, s, st);
    return rb ? norm_rows_launch<float, uint16_t, QUANT>(a, s, st)
              : norm_rows_launch<float, float, QUANT>(a, s, st);
  }
  if (!grid_x_fits(a.rows, kThreads)) return TCFP_ERR_SHAPE;
  norm_any_kernel<QUANT><<<unsigned(a.rows), kThreads, 0, st>>>(a);
  return launch_status();
}

}  // namespace

extern "C" {

int tcfp_rms_norm(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype,
                  int64_t ldr, const void* weight, int w_dtype, int64_t rows, int64_t cols,
                  float eps, void* h, void* y, int y_dtype, float* rstd, void* stream) {
  const Norm a{x, residual, weight, ldx, ldr, x_dtype, r_dtype, w_dtype, y_dtype, rows, cols,
               eps, 0, 0, 0, h, y, nullptr, nullptr, rstd};
  return norm_launch<false>(a, static_cast<hipStream_t>(stream));
}

int tcfp_rms_norm_quantize(const void* x, int x_dtype, int64_t ldx, const void* residual,
                           int r_dtype, int64_t ldr, const void* weight, int w_dtype,
                           int64_t rows, int64_t cols, float eps, int block, int fp8_fmt,
                           int f32_scales, void* h, uint8_t* q, void* scales, float* rstd,
                           void* stream) {
  const Norm a{x, residual, weight, ldx, ldr, x_dtype, r_dtype, w_dtype, 0, rows, cols,
               eps, block, fp8_fmt, f32_scales != 0, h, nullptr, q, scales, rstd};
  return norm_launch<true>(a, static_cast<hipStream_t>(stream));
}

size_t tcfp_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return size_t(parts_of(rows, cols)) * size_t(cols) * sizeof(float);
}

int tcfp_rms_norm_backward(const void* grad_y, int gy_dtype, const void* h, int h_dtype,
                           const float* rstd, const void* weight, int w_dtype,
                           const void* grad_h, int64_t rows, int64_t cols, void* dx, float* dw,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX) return TCFP_ERR_SHAPE;
  if (!dtype_ok(gy_dtype) || !dtype_ok(h_dtype) || !dtype_ok(w_dtype)) return TCFP_ERR_DTYPE;
  if (cols == 0 || (rows == 0 && !dw)) return TCFP_OK;
  const auto st = static_cast<hipStream_t>(stream);
  if (dw && rows > 0 && workspace_bytes < tcfp_rms_norm_backward_workspace_bytes(rows, cols))
    return TCFP_ERR_WORKSPACE;
  const int64_t parts = rows > 0 ? parts_of(rows, cols) : 0;
  // (one partial row is dw itself)
  NormBack a{grad_y, h, rstd, weight, grad_h, gy_dtype, h_dtype, w_dtype, rows, cols, dx,
             !dw ? nullptr : parts == 1 ? dw : static_cast<float*>(workspace)};
  if (rows > 0) {
    const RowShape s = back_shape(rows, cols);
    const bool vec = aligned(grad_y, 16) && aligned(h, 16) && aligned(weight, 16) &&
                     aligned(grad_h, 16) && aligned(dx, 16) && aligned(a.part, 16);
    if (s.t && vec) {
      const unsigned blocks = unsigned(
          dw ? parts : std::min<int64_t>((rows * s.t + wg_of(s.t) - 1) / wg_of(s.t), 2048));
      const bool gb = gy_dtype == TCFP_DTYPE_BF16, hb = h_dtype == TCFP_DTYPE_BF16;
      const bool nt = rows * cols * (size_of(gy_dtype) + (grad_h ? 2 : 1) * size_of(h_dtype)) >
                      kStreamBytes;
#define TCFP_NB_TYPES(NT)                                                          \
  do {                                                                             \
    if (gb && hb) norm_back_launch<uint16_t, uint16_t, NT>(a, s, blocks, st);      \
    else if (gb) norm_back_launch<uint16_t, float, NT>(a, s, blocks, st);          \
    else if (hb) norm_back_launch<float, uint16_t, NT>(a, s, blocks, st);          \
    else norm_back_launch<float, float, NT>(a, s, blocks, st);                     \
  } while (0)
      if (nt) TCFP_NB_TYPES(true);
      else TCFP_NB_TYPES(false);
#undef TCFP_NB_TYPES
    } else {
      if (!grid_x_fits(rows, kThreads)) return TCFP_ERR_SHAPE;
      norm_dx_any_kernel<<<unsigned(rows), kThreads, 0, st>>>(a);
      if (dw)
        norm_dw_any_kernel<<<dim3(unsigned((cols + kThreads - 1) / kThreads), unsigned(parts)),
                             kThreads, 0, st>>>(a, (rows + parts - 1) / parts);
    }
  }
  if (dw && parts != 1)
    norm_dw_sum_kernel<<<unsigned((cols + 15) / 16), kSumThreads, 0, st>>>(a.part, int(parts), cols,
                                                                        dw);
  return launch_status();
}

}  // extern "C"
