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

// The sum of v and the largest `top` over the THREADS threads of a row: a wavefront's lanes, or a workgroup of several
// wavefronts through `red` (used once).
struct Reduced {
  float sum;
  uint32_t top;
};
template <int THREADS>
__device__ __forceinline__ Reduced reduce_row(float v, uint32_t top, uint2 *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v += __shfl_xor(v, o);
    top = max(top, (uint32_t)__shfl_xor((int)top, o));
  }
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_uint2(__float_as_uint(v), top);
    __syncthreads();
    v = __uint_as_float(red[0].x);
    top = red[0].y;
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) {
      v += __uint_as_float(red[w].x);
      top = max(top, red[w].y);
    }
  }
  return Reduced{v, top};
}

// The same of sums in 64 bits.
template <int THREADS>
__device__ __forceinline__ double sum_row(double v, uint2 *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __builtin_bit_cast(uint2, v);
    __syncthreads();
    v = 0.;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += __builtin_bit_cast(double, red[w]);
  }
  return v;
}

// Eight int8 (KIND 1) or e4m3fn (KIND 2) codes of y * by, |y * by| at most the kind's largest number but for rounding.
template <int KIND>
__device__ __forceinline__ u32x2_t codes8(const float *y, float by) {
  float e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = y[j] * by;
  if constexpr (KIND == 1) {
    // 1.5 * 2^23 + e rounds e to a whole number, ties to even, whose low byte is the code
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(e[j] + 12582912.f);
    const uint32_t p0 = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), p1 = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    const uint32_t p2 = __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400), p3 = __builtin_amdgcn_perm(b[7], b[6], 0x04000c0c);
    return u32x2_t{p0 | p1, p2 | p3};
  } else {
    // v_cvt_pk_fp8_f32 rounds to nearest even and keeps subnormals: for every fp32 up to 448 the code of e4m3_code
    u32x2_t w = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = fminf(fmaxf(e[4 * h + j], -kF8Max), kF8Max);
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
      w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], x, true);
    }
    return w;
  }
}

// What turns a row into its norm and its codes. With z = t w and r = 1 / sqrt(mean(t^2) + eps), y = z r, and
// scale = max|z| r / q with q = 127 or 448: both reductions of a row are of its inputs alone and take one pass, and
// y / scale = z (q / max|z|). Each is the row's by one more rounding than (t r) w would take.
constexpr float kLeastMean = 0x1p-90f;  // below it the squares lose bits under fp32's smallest normal number
template <int KIND>
struct RowFactors {
  float y, code, scale;  // y: the factor r
  bool plain;          // else the squares or the products pass fp32 either way, or are not numbers
  __device__ __forceinline__ RowFactors(const Reduced &red, int hidden, float eps) {
    constexpr float kMost = KIND == 1 ? kI8Max : kF8Max;
    const float mean = red.sum / (float)hidden + eps;
    plain = mean > kLeastMean && red.sum < INFINITY && red.top < kInfBits;
    y = 1.f / sqrtf(mean);
    if constexpr (KIND != 0) {
      const float top = __uint_as_float(red.top), s = top * y / kMost;
      scale = fmaxf(s, 1e-12f);
      code = s > 1e-12f ? kMost / top : y / scale;
      plain = plain && top * y < INFINITY && code < INFINITY;
    }
  }
};

struct Rows {
  const uint16_t *x, *res, *w;
  int64_t x_row, res_row;
  void *out;
  float *scale;
  uint16_t *sum;
  int64_t out_row, sum_row;
  int rows, hidden;
  float eps;

  __device__ __forceinline__ void load(int64_t row, int c, float *t) const {
    unpack8r(ld16(x + row * x_row + 8 * c), t);
    if (res) {
      float b[8];
      unpack8r(ld16(res + row * res_row + 8 * c), b);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] += b[j];
    }
  }
  __device__ __forceinline__ void weights(int c, float *wf) const { unpack8r(ld16(w + 8 * c), wf); }
  // the outputs of chunk c: y is the norm (KIND 0), y * by the value that is coded
  template <int KIND>
  __device__ __forceinline__ void store(int64_t row, int c, const float *t, const float *y, float by) const {
    if constexpr (KIND == 0) {
      st16(static_cast<uint16_t *>(out) + row * out_row + 8 * c, pack8r(y));
    } else {
      *reinterpret_cast<u32x2_t *>(static_cast<uint8_t *>(out) + row * out_row + 8 * c) = codes8<KIND>(y, by);
    }
    // the next layer reads the sum, not the projection behind this kernel: it streams past the caches (253 -> 246 us below)
    if (sum) st16_stream(sum + row * sum_row + 8 * c, pack8r(t));
  }
};

// A row that fp32 does not hold that way, read and made once more: its squares, their sum, r and (t r) w in 64 bits, which
// hold them for any t and w (a power of two for the row would not do: t reaches from 2^-133 to 2^128, and what passed fp32 may
// be t w alone). A row whose y is not finite gets the scale NaN and zero codes. Loops over memory: the registers stay few.
template <int KIND, int THREADS>
__device__ __forceinline__ void norm_row_again(const Rows &p, int64_t row, int tid, uint2 (*red)[THREADS / 64]) {
  const int chunks = p.hidden / 8;
  asm volatile("" : "+v"(tid));  // no address of the ordinary pass is kept for this one
  double squares = 0.;
  float t[8], y[8];
#pragma unroll 1
  for (int c = tid; c < chunks; c += THREADS) {
    p.load(row, c, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) squares = fma((double)t[j], (double)t[j], squares);
  }
  const double r = 1. / sqrt(sum_row<THREADS>(squares, red[0]) / p.hidden + p.eps);
  auto normed = [&](int c) __device__ {
    p.load(row, c, t);
    p.weights(c, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)((double)t[j] * r * y[j]);
  };
  float by = 1.f;
  if constexpr (KIND != 0) {
    uint32_t top = 0;
#pragma unroll 1
    for (int c = tid; c < chunks; c += THREADS) {
      normed(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, abs_bits(y[j]));
    }
    top = reduce_row<THREADS>(0.f, top, red[1]).top;
    const float s = top < kInfBits ? fmaxf(__uint_as_float(top) / (KIND == 1 ? kI8Max : kF8Max), 1e-12f) : __builtin_nanf("");
    if (tid == 0) p.scale[row] = s;
    by = top < kInfBits ? 1.f / s : 0.f;
  }
#pragma unroll 1
  for (int c = tid; c < chunks; c += THREADS) {
    normed(c);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (KIND != 0 && by == 0.f) y[j] = 0.f;
    p.template store<KIND>(row, c, t, y, by);
  }
}

// One row on THREADS threads: `each` calls a function with every chunk of the row that the thread has (`tid`, tid + THREADS,
// ...) and its t. The outputs are written after every read of the row by another thread, each thread's over what it alone
// read, so the sum may lie over x or the residual.
template <int KIND, int THREADS, class Each>
__device__ __forceinline__ void norm_row(const Rows &p, int64_t row, int tid, uint2 (*red)[THREADS / 64], Each each) {
  float ss = 0.f;
  uint32_t top = 0;
  each([&](int c, const float *t) __device__ {
    float wf[8];
    if constexpr (KIND != 0) p.weights(c, wf);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(t[j], t[j], ss);
      if constexpr (KIND != 0) top = max(top, abs_bits(t[j] * wf[j]));
    }
  });
  const RowFactors<KIND> f(reduce_row<THREADS>(ss, top, red[0]), p.hidden, p.eps);
  if (!f.plain) return norm_row_again<KIND, THREADS>(p, row, tid, red + 1);
  if (KIND != 0 && tid == 0) p.scale[row] = f.scale;
  each([&](int c, const float *t) __device__ {
    float z[8];
    p.weights(c, z);
    // bf16: (t r) w, whose |t r| is at most sqrt(hidden); t w alone can pass fp32, and no reduction has looked at it
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] *= KIND == 0 ? t[j] * f.y : t[j];
    p.template store<KIND>(row, c, t, z, KIND == 0 ? 1.f : f.code);
  });
}

// Rows of up to 8 THREADS NCH channels: the row's sum stays in registers (fp32) from the loads, all in flight at once, to the
// outputs. THREADS 64: a wavefront per row, four rows per workgroup, no barrier; 256: a workgroup per row. Eight wavefronts a
// SIMD in bf16 (with six 20,000 rows x 2,048 take 49.5 us instead of 47.2; rows that are taken again spill 28 bytes then), six
// or more of the 8-bit kinds (with five x 2,560 in int8 took 73 instead of 69, x 5,120 127 instead of 125).
template <int KIND, int THREADS, int NCH>
__global__ __launch_bounds__(256, KIND ? 6 : 8) void residual_norm_kernel(Rows p) {
  __shared__ uint2 red[3][4];
  const int64_t row = THREADS == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= p.rows) return;  // a whole wavefront (THREADS 64) or none
  const int chunks = p.hidden / 8, tid = threadIdx.x % THREADS;
  u32x4_t xv[NCH], rv[NCH];
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    const int c = tid + THREADS * u;
    if (c < chunks) {
      xv[u] = ld16(p.x + row * p.x_row + 8 * c);
      if (p.res) rv[u] = ld16(p.res + row * p.res_row + 8 * c);
    }
  }
  float t[NCH][8];
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    if (tid + THREADS * u < chunks) {
      unpack8r(xv[u], t[u]);
      if (p.res) {
        float b[8];
        unpack8r(rv[u], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[u][j] += b[j];
      }
    }
  }
  norm_row<KIND, THREADS>(p, row, tid, reinterpret_cast<uint2 (*)[THREADS / 64]>(red), [&](auto f) __device__ {
#pragma unroll
    for (int u = 0; u < NCH; ++u)
      if (tid + THREADS * u < chunks) f(tid + THREADS * u, t[u]);
  });
}

// Longer rows: a workgroup per row that reads it once for the sums and once more for the outputs.
template <int KIND>
__global__ __launch_bounds__(256) void residual_norm_sweep_kernel(Rows p) {
  __shared__ uint2 red[3][4];
  const int64_t row = blockIdx.x;
  norm_row<KIND, 256>(p, row, threadIdx.x, red, [&](auto f) __device__ {
    for (int c = threadIdx.x; c < p.hidden / 8; c += 256) {
      float t[8];
      p.load(row, c, t);
      f(c, t);
    }
  });
}

// A workgroup per row, but for many narrow rows, which leave its threads one chunk each or less: a wavefront per row. 40,688
// rows x 5,120 in int8: 253 us against 282 with a wavefront and ten chunks a lane; x 2,048: 118 against 104, x 1,024: 93
// against 55. In bf16 the workgroup has less to do per row: x 2,048 113 against 117, x 1,024 68 against 53. 2,048 rows x 1,024
// in int8 6.9 against 5.6, 512 rows 3.5 against 3.8. HBM is the bound: 246 us for the 5,120 are 5.9 TB/s for the 7 bytes of
// an element, where a copy reaches 4.8.
constexpr int kWaveWidth = 2048, kWaveWidthBf16 = 1024, kWaveRows = 2048;

template <int KIND>
void launch_residual_norm(const Rows &p, hipStream_t s) {
  if (p.hidden > 8 * 256 * 4)
    hipLaunchKernelGGL(residual_norm_sweep_kernel<KIND>, dim3(p.rows), dim3(256), 0, s, p);
  else if (p.hidden <= (KIND ? kWaveWidth : kWaveWidthBf16) && p.rows >= kWaveRows)
    hipLaunchKernelGGL((residual_norm_kernel<KIND, 64, 4>), dim3((p.rows + 3) / 4), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((residual_norm_kernel<KIND, 256, 4>), dim3(p.rows), dim3(256), 0, s, p);
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
  if (rows == 1) x_row = residual_row = out_row = sum_row = hidden;  // one row has no stride, whatever a caller passes for it
  int rc = check_bf16_rows(x, x_row, hidden, "x", true);
  if (!rc && residual) rc = check_bf16_rows(residual, residual_row, hidden, "the residual", true);
  if (!rc) rc = check_bf16_rows(weight, hidden, hidden, "the weight");
  if (!rc && sum) rc = check_bf16_rows(sum, sum_row, hidden, "the sum");
  if (!rc && kind == 0) rc = check_bf16_rows(out, out_row, hidden, "out");
  if (!rc) rc = check_grid(rows, 256, "residual_rmsnorm");
  if (rc) return rc;
  if (kind != 0)
    VDNH3_HOST_CHECK(out && scale && out_row % 8 == 0 && out_row >= hidden && reinterpret_cast<uintptr_t>(out) % 8 == 0,
                     VDNH3_ERR_INVALID,
                     "residual_rmsnorm: codes must be 8-byte aligned with a row stride of a multiple of 8, and have scales");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Rows p{x, residual, weight, x_row, residual_row, out, scale, sum, out_row, sum_row, rows, hidden, eps};
  if (kind == 0) launch_residual_norm<0>(p, s);
  else if (kind == 1) launch_residual_norm<1>(p, s);
  else launch_residual_norm<2>(p, s);
  return check_launch("residual_rmsnorm");
}
