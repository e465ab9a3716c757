// Residual addition, RMSNorm and the activation quantisation of a W8A8 projection in one pass (HBM-bound):
//
//   t = x + residual                          stored as bf16(t), the residual stream of the next layer
//   y_j = t_j * r * w_j,  r = 1 / sqrt(mean(t^2) + eps)
//   bf16 : out = bf16(y)
//   int8 : scale = max(max|y| / 127, 1e-12), code = clamp(rne(y / scale), +-127)
//   e4m3 : scale = max(max|y| / 448, 1e-12), code = e4m3fn(clamp(y / scale, +-448))
//
// t, its sum of squares, y and the scale are fp32: the norm sees the sum before its rounding to bf16 and the codes
// see y before any, so every output is rounded once. A row whose y holds an infinity or a NaN (in the inputs, or a
// sum past fp32) gets the scale NaN and zero codes: every value that it stands for is NaN.
#include "common.h"

namespace vdnh3 {
namespace {

constexpr int kNormThreads = 256;

__device__ __forceinline__ void unpack8r(u32x4_t w, float *x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = w[j >> 1];
    x[j] = __uint_as_float((j & 1) ? (u & 0xffff0000u) : (u << 16));
  }
}

__device__ __forceinline__ u32x4_t pack8r(const float *y) {
  return u32x4_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7])};
}

// The bits of |y|: they order like the values, infinity above every number and a NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

// Sum / largest over a workgroup of WAVES wavefronts; `red` is used by one reduction only.
template <int WAVES>
__device__ __forceinline__ float workgroup_sum(float v, float *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += red[w];
  return s;
}
template <int WAVES>
__device__ __forceinline__ uint32_t workgroup_max(uint32_t v, uint32_t *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t m = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = max(m, red[w]);
  return m;
}

// The quantisation of a row whose largest |y| has the bits `top`.
template <int KIND>
struct RowScale {
  float s, r;
  bool fine;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    fine = top < kInfBits;
    s = fine ? fmaxf(__uint_as_float(top) / (KIND == 1 ? kI8Max : kF8Max), 1e-12f) : __builtin_nanf("");
    r = fine ? 1.f / s : 0.f;
  }
  // quant_div: y / s to within its last place, by a product and one correction
  __device__ __forceinline__ uint32_t code(float y) const {
    if (!fine) return 0;
    const float e = quant_div(y, s, r);
    return KIND == 1 ? i8_code(e) : e4m3_code(fminf(fmaxf(e, -kF8Max), kF8Max));
  }
  __device__ __forceinline__ u32x2_t codes(const float *y) const {
    u32x2_t w = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j >> 2] |= code(y[j]) << (8 * (j & 3));
    return w;
  }
};

// 1 / sqrt(mean + eps) from a row's sum of squares. A sum past fp32 (values above 1e19) is taken again from values
// scaled by 2^-64; `again` gives it.
template <class Again>
__device__ __forceinline__ float row_factor(float ss, int hidden, float eps, Again again) {
  if (ss < INFINITY) return 1.f / sqrtf(ss / (float)hidden + eps);
  constexpr float kDown = 5.421010862427522e-20f;  // 2^-64
  return kDown / sqrtf(again(kDown) / (float)hidden + eps * kDown * kDown);
}

// One workgroup per row, any width: a sweep over the row for the sum of squares, one for the largest |y| (8-bit
// kinds) and one for the outputs. The sum is written in the last sweep, each thread over what it alone read, so
// `sum` may be x or the residual itself.
template <int KIND>
__global__ __launch_bounds__(kNormThreads) void residual_norm_sweep_kernel(
    const uint16_t *x, int64_t x_row, const uint16_t *res, int64_t res_row, const uint16_t *__restrict__ w, float eps,
    int hidden, void *__restrict__ out, int64_t out_row, float *__restrict__ scale, uint16_t *sum, int64_t sum_row) {
  constexpr int WAVES = kNormThreads / 64;
  __shared__ float red[2][WAVES];
  __shared__ uint32_t top[WAVES];
  const int64_t row = blockIdx.x;
  const uint16_t *xr = x + row * x_row, *rr = res ? res + row * res_row : nullptr;
  const int chunks = hidden / 8;
  auto load = [&](int c, float *t) __device__ {
    unpack8r(ld16(xr + 8 * c), t);
    if (rr) {
      float b[8];
      unpack8r(ld16(rr + 8 * c), b);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] += b[j];
    }
  };
  auto squares = [&](float by, float *slot) __device__ {
    float ss = 0.f;
    for (int c = threadIdx.x; c < chunks; c += kNormThreads) {
      float t[8];
      load(c, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(t[j] * by, t[j] * by, ss);
    }
    return workgroup_sum<WAVES>(ss, slot);
  };
  const float r = row_factor(squares(1.f, red[0]), hidden, eps, [&](float by) __device__ { return squares(by, red[1]); });
  auto normed = [&](int c, const float *t, float *y) __device__ {
    float wf[8];
    unpack8r(ld16(w + 8 * c), wf);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = t[j] * r * wf[j];
  };
  uint32_t most = 0;
  if constexpr (KIND != 0) {
    for (int c = threadIdx.x; c < chunks; c += kNormThreads) {
      float t[8], y[8];
      load(c, t);
      normed(c, t, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, abs_bits(y[j]));
    }
    most = workgroup_max<WAVES>(most, top);
  }
  const RowScale<KIND> q(most);
  if (KIND != 0 && threadIdx.x == 0) scale[row] = q.s;
  for (int c = threadIdx.x; c < chunks; c += kNormThreads) {
    float t[8], y[8];
    load(c, t);
    normed(c, t, y);
    if constexpr (KIND == 0)
      st16(static_cast<uint16_t *>(out) + row * out_row + 8 * c, pack8r(y));
    else
      *reinterpret_cast<u32x2_t *>(static_cast<uint8_t *>(out) + row * out_row + 8 * c) = q.codes(y);
    if (sum) st16(sum + row * sum_row + 8 * c, pack8r(t));
  }
}

template <int KIND>
void launch_residual_norm(const uint16_t *x, int64_t x_row, const uint16_t *res, int64_t res_row, const uint16_t *w,
                          float eps, int rows, int hidden, void *out, int64_t out_row, float *scale, uint16_t *sum,
                          int64_t sum_row, hipStream_t s) {
  hipLaunchKernelGGL(residual_norm_sweep_kernel<KIND>, dim3(rows), dim3(kNormThreads), 0, s, x, x_row, res, res_row, w,
                     eps, hidden, out, out_row, scale, sum, sum_row);
}

// An operand that is only read may repeat one row (stride 0).
int check_bf16_rows(const void *p, int64_t row, int hidden, const char *name, bool read = false) {
  VDNH3_HOST_CHECK(p != nullptr && row % 8 == 0 && (row >= hidden || (read && row == 0)) && reinterpret_cast<uintptr_t>(p) % 16 == 0,
                   VDNH3_ERR_INVALID, "residual_rmsnorm: %s must be 16-byte aligned with a row stride of a multiple of 8 "
                   "that covers the width", name);
  return VDNH3_OK;
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_residual_rmsnorm_quant_rows(int kind, const uint16_t *x, int64_t x_row, const uint16_t *residual,
                                                 int64_t residual_row, const uint16_t *weight, float eps, int rows,
                                                 int hidden, void *out, int64_t out_row, float *scale, uint16_t *sum,
                                                 int64_t sum_row, void *stream) {
  using namespace vdnh3;
  VDNH3_HOST_CHECK(kind >= 0 && kind <= 2, VDNH3_ERR_INVALID,
                   "residual_rmsnorm: kind must be 0 (bf16), 1 (int8) or 2 (fp8), got %d", kind);
  VDNH3_HOST_CHECK(rows > 0 && hidden > 0 && hidden % 8 == 0, VDNH3_ERR_INVALID,
                   "residual_rmsnorm: rows must be positive and the width a positive multiple of 8, got %d x %d", rows,
                   hidden);
  VDNH3_HOST_CHECK(eps >= 0.f && eps < INFINITY, VDNH3_ERR_INVALID, "residual_rmsnorm: eps must be finite and not negative");
  int rc = check_bf16_rows(x, x_row, hidden, "x", true);
  if (!rc && residual) rc = check_bf16_rows(residual, residual_row, hidden, "the residual", true);
  if (!rc) rc = check_bf16_rows(weight, hidden, hidden, "the weight");
  if (!rc && sum) rc = check_bf16_rows(sum, sum_row, hidden, "the sum");
  if (!rc && kind == 0) rc = check_bf16_rows(out, out_row, hidden, "out");
  if (rc) return rc;
  if (kind != 0)
    VDNH3_HOST_CHECK(out && scale && out_row % 8 == 0 && out_row >= hidden && reinterpret_cast<uintptr_t>(out) % 8 == 0,
                     VDNH3_ERR_INVALID,
                     "residual_rmsnorm: codes must be 8-byte aligned with a row stride of a multiple of 8, and have scales");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (kind == 0)
    launch_residual_norm<0>(x, x_row, residual, residual_row, weight, eps, rows, hidden, out, out_row, scale, sum, sum_row, s);
  else if (kind == 1)
    launch_residual_norm<1>(x, x_row, residual, residual_row, weight, eps, rows, hidden, out, out_row, scale, sum, sum_row, s);
  else
    launch_residual_norm<2>(x, x_row, residual, residual_row, weight, eps, rows, hidden, out, out_row, scale, sum, sum_row, s);
  return check_launch("residual_rmsnorm");
}
