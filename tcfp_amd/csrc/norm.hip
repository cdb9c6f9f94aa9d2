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

enum { kPlain = 0, kExps = 1, kF32Scales = 2 };

struct Norm {
  const void* x;
  const void* r;
  const void* w;
  int64_t ldx, ldr;
  int x_dtype, r_dtype, w_dtype, y_dtype;
  int64_t rows;
  int64_t cols;
  float eps;
  int block, fmt;
  void* h;
  void* y;
  uint8_t* q;
  void* scales;
  float* rstd;
};

// One workgroup a row, any width and alignment: the row is read twice, the
// second time from L2.  Blocks of the quantised output are groups of 32
// consecutive threads, an element each, stepping over a block's columns.
template <int MODE>
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
  if constexpr (MODE == kPlain) {
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
      if constexpr (MODE == kF32Scales) {
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
        if constexpr (MODE == kF32Scales) static_cast<float*>(a.scales)[kb * a.rows + row] = inv;
        else static_cast<int8_t*>(a.scales)[kb * a.rows + row] = int8_t(e);
      }
    }
  }
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

__global__ __launch_bounds__(kThreads) void norm_dw_sum_kernel(const float* part, int64_t parts,
                                                               int64_t cols, float* dw) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int64_t p = 0; p < parts; ++p) s += part[p * cols + c];
  dw[c] = s;
}

constexpr int64_t kMaxParts = 256;

int norm_checks(const Norm& a, bool quantised) {
  if (a.rows < 0 || a.cols < 0 || a.rows > INT32_MAX || a.cols > INT32_MAX) return TCFP_ERR_SHAPE;
  if (a.ldx < a.cols || (a.r && a.ldr < a.cols)) return TCFP_ERR_SHAPE;
  if (!dtype_ok(a.x_dtype) || !dtype_ok(a.w_dtype) || (a.r && !dtype_ok(a.r_dtype)))
    return TCFP_ERR_DTYPE;
  if (a.h && !a.r) return TCFP_ERR_SHAPE;
  if (!grid_x_fits(a.rows, kThreads)) return TCFP_ERR_SHAPE;
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

template <int MODE>
int norm_launch(const Norm& a, hipStream_t st) {
  const int rc = norm_checks(a, MODE != kPlain);
  if (rc != TCFP_OK || a.rows == 0 || a.cols == 0) return rc;
  norm_any_kernel<MODE><<<unsigned(a.rows), kThreads, 0, st>>>(a);
  return launch_status();
}

}  // namespace

extern "C" {

int tcfp_rms_norm(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype,
                  int64_t ldr, const void* weight, int w_dtype, int64_t rows, int64_t cols,
                  float eps, void* h, void* y, int y_dtype, float* rstd, void* stream) {
  const Norm a{x, residual, weight, ldx, ldr, x_dtype, r_dtype, w_dtype, y_dtype, rows, cols,
               eps, 0, 0, h, y, nullptr, nullptr, rstd};
  return norm_launch<kPlain>(a, static_cast<hipStream_t>(stream));
}

int tcfp_rms_norm_quantize(const void* x, int x_dtype, int64_t ldx, const void* residual,
                           int r_dtype, int64_t ldr, const void* weight, int w_dtype,
                           int64_t rows, int64_t cols, float eps, int block, int fp8_fmt,
                           int f32_scales, void* h, uint8_t* q, void* scales, float* rstd,
                           void* stream) {
  const Norm a{x, residual, weight, ldx, ldr, x_dtype, r_dtype, w_dtype, 0, rows, cols,
               eps, block, fp8_fmt, h, nullptr, q, scales, rstd};
  const auto st = static_cast<hipStream_t>(stream);
  return f32_scales ? norm_launch<kF32Scales>(a, st) : norm_launch<kExps>(a, st);
}

size_t tcfp_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return size_t(std::min(rows, kMaxParts)) * size_t(cols) * sizeof(float);
}

int tcfp_rms_norm_backward(const void* grad_y, int gy_dtype, const void* h, int h_dtype,
                           const float* rstd, const void* weight, int w_dtype,
                           const void* grad_h, int64_t rows, int64_t cols, void* dx, float* dw,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX) return TCFP_ERR_SHAPE;
  if (!grid_x_fits(rows, kThreads)) return TCFP_ERR_SHAPE;
  if (!dtype_ok(gy_dtype) || !dtype_ok(h_dtype) || !dtype_ok(w_dtype)) return TCFP_ERR_DTYPE;
  if (cols == 0 || (rows == 0 && !dw)) return TCFP_OK;
  const auto st = static_cast<hipStream_t>(stream);
  const unsigned cg = unsigned((cols + kThreads - 1) / kThreads);
  if (dw && workspace_bytes < tcfp_rms_norm_backward_workspace_bytes(rows, cols))
    return TCFP_ERR_WORKSPACE;
  const NormBack a{grad_y, h, rstd, weight, grad_h, gy_dtype, h_dtype, w_dtype, rows, cols,
                   dx, static_cast<float*>(workspace)};
  if (rows > 0) norm_dx_any_kernel<<<unsigned(rows), kThreads, 0, st>>>(a);
  if (dw) {
    const int64_t parts = std::min(rows, kMaxParts);
    if (rows > 0) {
      const int64_t per = (rows + parts - 1) / parts;
      norm_dw_any_kernel<<<dim3(cg, unsigned(parts)), kThreads, 0, st>>>(a, per);
    }
    norm_dw_sum_kernel<<<cg, kThreads, 0, st>>>(a.part, parts, cols, dw);
  }
  return launch_status();
}

}  // extern "C"
