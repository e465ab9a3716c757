// q / k RMSNorm (optional) and the rotary embedding of positions on several axes (HBM-bound):
//
//   y_d = x_d * r * w_d (with weights; y = x without), the arithmetic of qk_norm.h
//   pair i of rot / 2 turns by angle_i = 2 pi * position[axis_i][row] * turns_i:
//   out_i = y_i cos - y_{i+h} sin,  out_{i+h} = y_i sin + y_{i+h} cos,  h = rot / 2; channels >= rot pass
//
// position * turns is taken in 64 bits and only its fraction rounded to fp32: at position 40,688 an fp32 angle would be
// off by 2e-3, a bf16 step. q and k have their own numbers of heads; one rounding to bf16 at the end.
#include "common.h"
#include "qk_norm.h"

namespace vdnh3 {
namespace {

struct Positions {
  const void *p;
  int64_t axis, row;  // strides
  int type;           // 0 int32, 1 int64, 2 fp32
};

__device__ __forceinline__ double position_at(const Positions &pos, int axis, int64_t row) {
  const int64_t at = axis * pos.axis + row * pos.row;
  if (pos.type == 0) return (double)static_cast<const int32_t *>(pos.p)[at];
  if (pos.type == 1) return (double)static_cast<const int64_t *>(pos.p)[at];
  return (double)static_cast<const float *>(pos.p)[at];
}

// cos and sin of 2 pi times the fraction of position * turns
__device__ __forceinline__ float2 turn(double position, double turns) {
  const double t = position * turns;
  float s, c;
  sincospif(2.f * (float)(t - rint(t)), &s, &c);
  return make_float2(c, s);
}

struct Vectors {
  const uint16_t *x;
  int64_t row, head;
  const uint16_t *w;
  float eps;
  uint16_t *out;
  int64_t out_row, out_head;
  int heads;
};

// One group of LANES lanes per head vector, 8 channels a lane; dim <= 8 LANES, lanes past it idle.
template <int LANES>
__global__ __launch_bounds__(256) void rotary_kernel(Vectors q, Vectors k, Positions pos,
                                                     const double *__restrict__ turns, const int32_t *__restrict__ axis,
                                                     int rot, int dim, int64_t n_vec) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t vec = t / LANES;
  const int c = (int)(t % LANES);
  if (vec >= n_vec) return;  // a lane group is wholly in range or wholly out
  const int nv = q.heads + k.heads;
  const int64_t row = vec / nv;
  const int v = (int)(vec - row * nv), which = v >= q.heads, head = which ? v - q.heads : v;
  const Vectors &s = which ? k : q;
  const bool live = 8 * c < dim;
  float y[8] = {}, o[8];
  if (live) {
    const u32x4_t raw = ld16(s.x + row * s.row + head * s.head + 8 * c);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = __uint_as_float((j & 1) ? (raw[j >> 1] & 0xffff0000u) : (raw[j >> 1] << 16));
  }
  if (s.w) {
    const float r = rms_factor(group_tree_sum<LANES>(chunk_sumsq(y)), dim, s.eps);
    if (live) {
      const u32x4_t w = ld16(s.w + 8 * c);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y[j] = y[j] * r * __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
    }
  }
  const int half = rot >> 1, step = half >> 3, lane = __lane_id();
  const bool first = 8 * c < half, rotated = 8 * c < rot;
  const int partner = !rotated ? lane : first ? lane + step : lane - step;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = __shfl(y[j], partner);
  if (!live) return;
  if (rotated) {
    const int i0 = first ? 8 * c : 8 * c - half;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 cs = turn(position_at(pos, axis[i0 + j], row), turns[i0 + j]);
      y[j] = rope_rotate(y[j], o[j], f32x4_t{cs.x, -cs.y, cs.y, cs.x}, first);
    }
  }
  st16(s.out + row * s.out_row + head * s.out_head + 8 * c,
       u32x4_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7])});
}

int check_vectors(const Vectors &s, const char *name) {
  VDNH3_HOST_CHECK(s.x && s.out, VDNH3_ERR_INVALID, "rotary: %s or its output is null", name);
  VDNH3_HOST_CHECK(s.row % 8 == 0 && s.head % 8 == 0 && s.out_row % 8 == 0 && s.out_head % 8 == 0 &&
                       (reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.out) |
                        reinterpret_cast<uintptr_t>(s.w)) % 16 == 0,
                   VDNH3_ERR_INVALID,
                   "rotary: %s, its output and its weight must be 16-byte aligned with strides that are multiples of 8", name);
  return VDNH3_OK;
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_qk_rotary_axes(const uint16_t *q, int64_t q_row, int64_t q_head, const uint16_t *q_weight, float q_eps,
                                    uint16_t *q_out, int64_t qo_row, int64_t qo_head, int q_heads, const uint16_t *k,
                                    int64_t k_row, int64_t k_head, const uint16_t *k_weight, float k_eps, uint16_t *k_out,
                                    int64_t ko_row, int64_t ko_head, int k_heads, const void *positions, int position_type,
                                    int64_t p_axis, int64_t p_row, const double *turns, const int32_t *axis_of_pair,
                                    int rot_dim, int rows, int head_dim, void *stream) {
  using namespace vdnh3;
  VDNH3_HOST_CHECK(head_dim > 0 && head_dim <= 128 && head_dim % 8 == 0, VDNH3_ERR_INVALID,
                   "rotary: head_dim must be a multiple of 8 up to 128, got %d", head_dim);
  VDNH3_HOST_CHECK(rot_dim > 0 && rot_dim % 16 == 0 && rot_dim <= head_dim, VDNH3_ERR_INVALID,
                   "rotary: rot_dim must be a positive multiple of 16 and at most head_dim %d, got %d", head_dim, rot_dim);
  VDNH3_HOST_CHECK(rows > 0 && q_heads > 0 && k_heads > 0, VDNH3_ERR_INVALID, "rotary: rows and heads must be positive");
  VDNH3_HOST_CHECK(positions && turns && axis_of_pair && position_type >= 0 && position_type <= 2, VDNH3_ERR_INVALID,
                   "rotary: null positions or frequencies, or a position type other than 0 (int32), 1 (int64), 2 (fp32)");
  const Vectors qs{q, q_row, q_head, q_weight, q_eps, q_out, qo_row, qo_head, q_heads};
  const Vectors ks{k, k_row, k_head, k_weight, k_eps, k_out, ko_row, ko_head, k_heads};
  int rc = check_vectors(qs, "q");
  if (!rc) rc = check_vectors(ks, "k");
  if (rc) return rc;
  const Positions pos{positions, p_axis, p_row, position_type};
  const int64_t n_vec = (int64_t)rows * (q_heads + k_heads);
  const int lanes = head_dim <= 64 ? 8 : 16;
  const int64_t groups = (n_vec * lanes + 255) / 256;
  VDNH3_HOST_CHECK(groups <= INT32_MAX, VDNH3_ERR_INVALID, "rotary: %lld head vectors are too many for one launch",
                   (long long)n_vec);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (lanes == 8)
    hipLaunchKernelGGL(rotary_kernel<8>, dim3((unsigned)groups), dim3(256), 0, s, qs, ks, pos, turns, axis_of_pair, rot_dim,
                       head_dim, n_vec);
  else
    hipLaunchKernelGGL(rotary_kernel<16>, dim3((unsigned)groups), dim3(256), 0, s, qs, ks, pos, turns, axis_of_pair, rot_dim,
                       head_dim, n_vec);
  return check_launch("rotary");
}
