// q / k RMSNorm (optional) and the rotary embedding of positions on several axes (HBM-bound):
//
//   y_d = x_d * r * w_d (with weights; y = x without), the arithmetic of qk_norm.h; in 64 bits for vectors whose squares leave fp32
//   pair i of rot / 2 turns by angle_i = 2 pi * position[axis_i][row] * turns_i:
//   out_i = y_i cos - y_{i+h} sin,  out_{i+h} = y_i sin + y_{i+h} cos,  h = rot / 2; channels >= rot pass
//
// A workgroup computes its rows' angles itself: a table of rotations would be 16 more bytes a row and pair to write and read.
// position * turns is taken in 64 bits and only its fraction rounded to fp32: at position 40,688 an fp32 angle would be off
// by 2e-3, a bf16 step. q and k have their own numbers of heads; one rounding to bf16 at the end.
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

// The vectors of one row's q or k that a lane group takes: heads j, j + step, ... (its 8 channels of each), RB of them in
// flight. cs holds cos and sin of the lane's pairs, the second of a pair with the sine's sign turned.
template <int LANES, int RB>
__device__ __forceinline__ void turn_heads(const Vectors &s, int64_t row, int j, int step, int c, int dim, bool rotated,
                                           bool row_turn, int partner, const float2 (&cs)[8]) {
  // of a mean below 2^-90 the squares fall under what fp32 holds with all bits
  constexpr float kMostFactor = 0x1p45f;
  const bool live = 8 * c < dim;
  const uint16_t *x = s.x + row * s.row + 8 * c;
  uint16_t *out = s.out + row * s.out_row + 8 * c;
  float wf[8];
  if (s.w && live) {
    const u32x4_t w = ld16(s.w + 8 * c);
#pragma unroll
    for (int i = 0; i < 8; ++i) wf[i] = __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
  }
  // the turn of a normalised vector, and its store
  auto finish = [&](float (&y)[8], int h, bool keep) __device__ {
    float o[8];
    if (row_turn) {  // the partner is 8 lanes away in a 16-lane DPP row (row_ror:8)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o[i] = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y[i]), 0x128, 0xf, 0xf, false));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __shfl(y[i], partner);
    }
    if (rotated) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fmaf(cs[i].x, y[i], cs[i].y * o[i]);
    }
    if (live && keep)
      st16(out + h * s.out_head,
           u32x4_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7])});
  };
  auto unpack = [&](const u32x4_t &raw, float (&y)[8]) __device__ {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __uint_as_float((i & 1) ? (raw[i >> 1] & 0xffff0000u) : (raw[i >> 1] << 16));
  };
  bool again = false;
  for (int h0 = j; h0 < s.heads; h0 += RB * step) {
    u32x4_t raw[RB];
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      raw[u] = u32x4_t{0, 0, 0, 0};
      if (live && h0 + u * step < s.heads) raw[u] = ld16(x + (h0 + u * step) * s.head);
    }
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      if (h0 + u * step >= s.heads) break;  // a whole lane group
      float y[8];
      unpack(raw[u], y);
      bool fits = true;
      if (s.w) {
        const float ss = group_tree_sum<LANES>(chunk_sumsq(y)), r = rms_factor(ss, dim, s.eps);
        fits = r < kMostFactor && ss < INFINITY;
        again = again || !fits;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * r * wf[i];
      }
      finish(y, h0 + u * step, fits);
    }
  }
  if (!again) return;
  // Vectors whose squares fp32 does not hold, the norm in 64 bits: in a loop of their own, since in the one above its registers
  // took a wavefront a SIMD (of contiguous operands 40,688 rows x 80 heads take 306.6 us this way, 305.6 without; 512 x 48 6.6
  // and 6.4).
#pragma unroll 1
  for (int h = j; h < s.heads; h += step) {
    float y[8];
    unpack(live ? ld16(x + h * s.head) : u32x4_t{0, 0, 0, 0}, y);
    const float fp32 = group_tree_sum<LANES>(chunk_sumsq(y));
    if (rms_factor(fp32, dim, s.eps) < kMostFactor && fp32 < INFINITY) continue;  // a whole lane group
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma((double)y[i], (double)y[i], ss);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor(ss, o);
    const double r = 1. / sqrt(ss / dim + s.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)(y[i] * r * wf[i]);
    finish(y, h, true);
  }
}

// A workgroup takes R rows: its threads compute the rows' cosines and sines once, one pair each (R rot / 2 <= 256 at the
// widths that R is made for), and share them through LDS. LANES lanes hold a head vector, 8 channels each (dim <= 8 LANES,
// lanes past it idle), 256 / LANES / R lane groups a row; a group keeps its row's pairs in registers and walks the heads.
template <int LANES, int R>
__global__ __launch_bounds__(256, LANES == 16 ? 5 : 4) void rotary_kernel(Vectors q, Vectors k, Positions pos,
                                                                          const double *__restrict__ turns,
                                                                          const int32_t *__restrict__ axis, int rot, int dim,
                                                                          int rows) {
  constexpr int PAIRS = 4 * LANES, STEP = 256 / LANES / R;
  __shared__ __attribute__((aligned(16))) float2 table[R][PAIRS];
  const int half = rot >> 1, tid = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * R;
  for (int i = tid; i < R * PAIRS; i += 256) {
    const int r = i / PAIRS, pair = i % PAIRS;
    if (pair < half && row0 + r < rows) table[r][pair] = turn(position_at(pos, axis[pair], row0 + r), turns[pair]);
  }
  __syncthreads();
  const int c = tid % LANES, group = tid / LANES, r = group % R, j = group / R;
  const int64_t row = row0 + r;
  if (row >= rows) return;  // a whole lane group
  const bool first = 8 * c < half, rotated = 8 * c < rot;
  const int lane = __lane_id(), partner = !rotated ? lane : first ? lane + (half >> 3) : lane - (half >> 3);
  float2 cs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = table[r][rotated ? (first ? 8 * c : 8 * c - half) + i : 0];
    cs[i] = make_float2(f.x, first ? -f.y : f.y);
  }
  const bool row_turn = LANES == 16 && rot == 128;
  turn_heads<LANES, 4>(q, row, j, STEP, c, dim, rotated, row_turn, partner, cs);
  turn_heads<LANES, 4>(k, row, j, STEP, c, dim, rotated, row_turn, partner, cs);
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

// Rows of a workgroup: as few as keep the launch within one round, 4 workgroups a CU; more rows share a workgroup's other
// threads for the angles. 40 + 8 heads of 128: 512 rows 7.8 us (1 row), 9.0 (2), 12.3 (4); 2,048 rows 15.3, 13.8, 15.5; 4,096
// rows 30, 27, 23; 32 + 8 heads of 64: 2,048 rows 10.5, 8.1, 11.0 (8). HBM is the bound of many rows: 40,688 x 80 heads x 128
// take 327 us with the norms, 5.1 TB/s; 2 or 8 vectors in flight instead of 4 and non-temporal loads are no faster.
constexpr int kRound = 1024;

template <int LANES, int R>
void launch_rotary(const Vectors &q, const Vectors &k, const Positions &pos, const double *turns, const int32_t *axis, int rot,
                   int dim, int rows, hipStream_t s) {
  if constexpr (R < 64 / LANES) {  // at most a pair per thread
    if (rows > R * kRound) return launch_rotary<LANES, 2 * R>(q, k, pos, turns, axis, rot, dim, rows, s);
  }
  hipLaunchKernelGGL((rotary_kernel<LANES, R>), dim3((rows + R - 1) / R), dim3(256), 0, s, q, k, pos, turns, axis, rot, dim,
                     rows);
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
  VDNH3_HOST_CHECK(q_eps >= 0.f && k_eps >= 0.f && q_eps < INFINITY && k_eps < INFINITY, VDNH3_ERR_INVALID,
                   "rotary: eps must be finite and not negative");
  VDNH3_HOST_CHECK(rows > 0 && q_heads > 0 && k_heads > 0, VDNH3_ERR_INVALID, "rotary: rows and heads must be positive");
  VDNH3_HOST_CHECK(positions && turns && axis_of_pair && position_type >= 0 && position_type <= 2, VDNH3_ERR_INVALID,
                   "rotary: null positions or frequencies, or a position type other than 0 (int32), 1 (int64), 2 (fp32)");
  // a dimension of one element has no stride, whatever a caller passes for it
  auto stride = [](int64_t s, int extent) { return extent > 1 ? s : 0; };
  const Vectors qs{q, stride(q_row, rows), stride(q_head, q_heads), q_weight, q_eps, q_out, stride(qo_row, rows),
                   stride(qo_head, q_heads), q_heads};
  const Vectors ks{k, stride(k_row, rows), stride(k_head, k_heads), k_weight, k_eps, k_out, stride(ko_row, rows),
                   stride(ko_head, k_heads), k_heads};
  int rc = check_vectors(qs, "q");
  if (!rc) rc = check_vectors(ks, "k");
  if (!rc) rc = check_grid(rows, 64, "rotary");  // four rows a workgroup of 256 threads or more, or few rows
  if (rc) return rc;
  const Positions pos{positions, p_axis, p_row, position_type};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim <= 64)
    launch_rotary<8, 1>(qs, ks, pos, turns, axis_of_pair, rot_dim, head_dim, rows, s);
  else
    launch_rotary<16, 1>(qs, ks, pos, turns, axis_of_pair, rot_dim, head_dim, rows, s);
  return check_launch("rotary");
}
