// New tokens over the requests' recurrent states on gfx950: the single-token forms of the linear attention with a decay for
// each head (prompts: causal_linear.hip) and of the Gated DeltaNet (prompts: gdn.hip). Per value head, S [dv, dk] in fp32:
//
//   linear:  S_t = a_h S_{t-1} + v_t k_t^T,                            o_t = scale S_t q_t,   a_h = exp(log_decay_h)
//   delta:   S_t = a_t S_{t-1} (I - b_t k_t k_t^T) + b_t v_t k_t^T,    o_t = S_t q_t,         a_t = exp(g_t)
//          = a_t S_{t-1} + b_t (v_t - a_t S_{t-1} k_t) k_t^T
//
// Request b's states are pool[slots[b]]; they are read once, taken through the call's tokens in registers and written once.
// The rows of S do not see each other, so that they divide over wavefronts and workgroups freely.
#include <cmath>

#include "common.h"

namespace vdnh3 {
namespace {

struct StepRows {
  const uint16_t *p;
  int64_t batch, row, head;
};
struct StepGates {
  const float *p;
  int64_t batch, row, head;
};

struct StepCall {
  StepRows q, k, v;
  uint16_t *out;
  int64_t o_batch, o_row, o_head;
  const float *log_decay;  // linear: one per head
  StepGates beta, g;       // delta
  float *pool;
  int64_t slot_stride, head_stride;
  const int32_t *slots;
  int slot_count, tokens, heads, group, dim, parts;
  float scale;
};

// x summed over the 16 lanes of a row of the wavefront, in every one of them (row_ror: rotations inside a row)
template <int N>
__device__ __forceinline__ float rotated(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum16(float x) {
  x += rotated<8>(x);
  x += rotated<4>(x);
  x += rotated<2>(x);
  x += rotated<1>(x);
  return x;
}

// Columns of a row of the state: lane l16 has 4 l16 .. + 3 of each 64. The last of a head dim that is no multiple of 64 are
// left out.
template <bool VEC, bool STREAM>
__device__ __forceinline__ f32x4_t load4(const float *p, int c, int dim) {
  if constexpr (VEC) {
    const f32x4_t *at = reinterpret_cast<const f32x4_t *>(p + c);
    return c >= dim ? f32x4_t{} : STREAM ? __builtin_nontemporal_load(at) : *at;
  } else {
    f32x4_t x = {};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < dim) x[j] = p[c + j];
    return x;
  }
}
template <bool VEC, bool STREAM>
__device__ __forceinline__ void store4(float *p, int c, int dim, f32x4_t x) {
  if constexpr (VEC) {
    f32x4_t *at = reinterpret_cast<f32x4_t *>(p + c);
    if (c >= dim) return;
    if (STREAM) __builtin_nontemporal_store(x, at);
    else *at = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < dim) p[c + j] = x[j];
  }
}
template <bool VEC>
__device__ __forceinline__ f32x4_t load4(const uint16_t *p, int c, int dim) {
  f32x4_t x = {};
  if constexpr (VEC) {
    if (c < dim) {
      const u32x2_t w = *reinterpret_cast<const u32x2_t *>(p + c);
      x = f32x4_t{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                  __uint_as_float(w[1] & 0xffff0000u)};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < dim) x[j] = bf2f(p[c + j]);
  }
  return x;
}

// MODE 0: any layout and head dim, number by number; 1: 16-byte columns; 2: the same, and the head dim is the lanes' 16 E.
// A workgroup takes 16 G rows of one request's state of one head: a wavefront 4 G of them, 16 lanes a row, E columns a lane.
// HBM is the bound: 64 requests x 40 heads x 128 (335 MB) take 61.5 us, 5.5 TB/s, where a large copy reaches 4.8; one request
// 4.5 us, a launch and two chains of loads. 32 rows a workgroup (with states in the caches 65 us, 16 rows 74, 64 rows 69, 128
// rows 79; one request 4.5, 4.2, 5.3, 7.2). States of more than 64 channels pass the caches both ways: between two tokens lie the
// other layers' states (70.7 us without, 67 read so, 68.6 written so; a state that is still in the caches 60.8, and 58.6 read
// so; of 64 channels 25.3, and 23.1 without either if it is there). Several tokens of a request follow one another through its
// state, each a chain of its own loads, products and lane sums: 16 requests x 32 heads x 64 take 5.2 us for one token, 7.4 for four
// and 14.3 for eight (delta 5.5, 8.5, 15.7), 64 x 40 x 128 59, 81 and 118 (58, 87, 134).
template <bool DELTA, int E, int G, int MODE>
__global__ __launch_bounds__(256) void state_step_kernel(StepCall p) {
  constexpr int Q = E / 4;
  constexpr bool VEC = MODE > 0;
  const int part = (int)blockIdx.x % p.parts, rest = (int)blockIdx.x / p.parts, h = rest % p.heads, b = rest / p.heads;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, r4 = lane >> 4;
  const int row0 = (part * 4 + (tid >> 6)) * 4 * G;  // the wavefront's first row
  const int dim = p.dim;

  const int slot = p.slots ? p.slots[b] : b;
  const bool live = slot >= 0 && slot < p.slot_count;
  f32x4_t s[G][Q];
  float *state = p.pool + (live ? slot * p.slot_stride : 0) + h * p.head_stride;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = row0 + 4 * g + r4;
#pragma unroll
    for (int c = 0; c < Q; ++c)
      s[g][c] = live && r < dim ? load4<VEC, (E > 4)>(state + (int64_t)r * dim, 64 * c + 4 * l16, dim) : f32x4_t{};
  }
  // one request a slot: the first that names it has it, whatever order the workgroups run in
  bool taken = false;
  if (p.slots)
    for (int i = lane; i - lane < b; i += 64) taken = taken || __any(i < b && p.slots[i] == slot);

  const int hk = h / p.group;
  const uint16_t *qp = p.q.p + b * p.q.batch + hk * p.q.head, *kp = p.k.p + b * p.k.batch + hk * p.k.head;
  const uint16_t *vp = p.v.p + b * p.v.batch + h * p.v.head;
  uint16_t *op = p.out + b * p.o_batch + h * p.o_head;
  float a = DELTA ? 0.f : expf(p.log_decay[h]), beta = 0.f;
  for (int t = 0; t < p.tokens; ++t) {
    f32x4_t q[Q], k[Q];
#pragma unroll
    for (int c = 0; c < Q; ++c) {
      q[c] = load4<VEC>(qp + t * p.q.row, 64 * c + 4 * l16, dim);
      k[c] = load4<VEC>(kp + t * p.k.row, 64 * c + 4 * l16, dim);
    }
    if (DELTA) {
      a = expf(p.g.p[b * p.g.batch + t * p.g.row + h * p.g.head]);
      beta = p.beta.p[b * p.beta.batch + t * p.beta.row + h * p.beta.head];
    }
    float o = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int r = row0 + 4 * g + r4;
      float u = r < dim ? bf2f(vp[t * p.v.row + r]) : 0.f;
      if (DELTA) {
        float sk = 0.f;
#pragma unroll
        for (int c = 0; c < Q; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) sk = fmaf(s[g][c][j], k[c][j], sk);
        u = beta * fmaf(-a, sum16(sk), u);
      }
      float dot = 0.f;
#pragma unroll
      for (int c = 0; c < Q; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[g][c][j] = fmaf(a, s[g][c][j], u * k[c][j]);
          // columns behind the head dim stay zeros, also where u is no finite number
          if (MODE < 2 && 64 * c + 4 * l16 + j >= dim) s[g][c][j] = 0.f;
          dot = fmaf(s[g][c][j], q[c][j], dot);
        }
      dot = sum16(dot);
      if (l16 == g) o = dot;  // G is at most 16: lane g of a row's 16 keeps group g's
    }
    const int r = row0 + 4 * l16 + r4;
    if (l16 < G && r < dim) op[t * p.o_row + r] = f2bf(!live ? 0.f : taken ? __builtin_nanf("") : DELTA ? o : o * p.scale);
  }
  if (!live || taken) return;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = row0 + 4 * g + r4;
    if (r < dim)
#pragma unroll
      for (int c = 0; c < Q; ++c) store4<VEC, (E > 4)>(state + (int64_t)r * dim, 64 * c + 4 * l16, dim, s[g][c]);
  }
}

template <bool DELTA, int MODE>
void launch_state_step(StepCall p, int batch, hipStream_t s) {
  auto run = [&](auto kernel, int rows) {
    p.parts = (p.dim + rows - 1) / rows;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)p.parts * p.heads * batch)), dim3(256), 0, s, p);
  };
  if (p.dim > 64) run(state_step_kernel<DELTA, 8, 2, MODE>, 32);
  else run(state_step_kernel<DELTA, 4, 2, MODE>, 32);
}

bool fits4(const void *p, int64_t a, int64_t b, int64_t c, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && a % 4 == 0 && b % 4 == 0 && c % 4 == 0;
}

template <bool DELTA>
int state_step(const uint16_t *q, const uint16_t *k, const uint16_t *v, uint16_t *out, const float *decay, const float *beta,
               float *pool, const int32_t *slots, const vdnh3_step_layout *layout, float scale, void *stream, const char *what) {
  VDNH3_HOST_CHECK(layout != nullptr, VDNH3_ERR_INVALID, "%s: a layout is needed", what);
  const vdnh3_step_layout &l = *layout;
  for (const int64_t n : {l.slots, l.batch, l.new_tokens, l.heads, l.qk_heads, l.head_dim})
    VDNH3_HOST_CHECK(n > 0 && n <= INT32_MAX, VDNH3_ERR_INVALID, "%s: sizes must be positive and fit 32 bits, got %lld", what,
                     (long long)n);
  VDNH3_HOST_CHECK(l.heads % l.qk_heads == 0, VDNH3_ERR_INVALID, "%s: %lld heads are no multiple of %lld q / k heads", what,
                   (long long)l.heads, (long long)l.qk_heads);
  VDNH3_HOST_CHECK(l.head_dim <= 128, VDNH3_ERR_INVALID, "%s: head_dim must be 1 to 128, got %lld", what, (long long)l.head_dim);
  VDNH3_HOST_CHECK(q && k && v && out && pool && decay && (beta || !DELTA), VDNH3_ERR_INVALID, "%s: an operand is missing", what);
  VDNH3_HOST_CHECK(slots || l.batch <= l.slots, VDNH3_ERR_INVALID, "%s: %lld requests need a state each, the pool has %lld", what,
                   (long long)l.batch, (long long)l.slots);
  const int64_t own = l.head_dim * l.head_dim;
  // one state behind another, heads inside slots or slots inside heads; a stride of a single one is not looked at
  auto apart = [own](int64_t inner, int64_t count, int64_t outer) {
    return inner >= own && inner <= (INT64_MAX >> 32) && outer >= (count - 1) * inner + own;
  };
  VDNH3_HOST_CHECK(l.heads == 1 || l.slots == 1
                       ? (l.slots == 1 || l.slot >= own) && (l.heads == 1 || l.state_head >= own)
                       : apart(l.state_head, l.heads, l.slot) || apart(l.slot, l.slots, l.state_head),
                   VDNH3_ERR_INVALID, "%s: states must not overlap", what);
  VDNH3_HOST_CHECK(std::isfinite(scale), VDNH3_ERR_INVALID, "%s: scale must be finite", what);
  const int64_t per_request = (l.head_dim + 31) / 32 * l.heads;
  const int rc = check_grid(per_request > (1 << 24) ? per_request : per_request * l.batch, 256, what);
  if (rc) return rc;
  const StepCall p{{q, l.q_batch, l.q_row, l.q_head}, {k, l.k_batch, l.k_row, l.k_head}, {v, l.v_batch, l.v_row, l.v_head},
                   out, l.o_batch, l.o_row, l.o_head, decay, {beta, l.beta_batch, l.beta_row, l.beta_head},
                   {decay, l.g_batch, l.g_row, l.g_head}, pool, l.slot, l.state_head, slots, (int)l.slots, (int)l.new_tokens,
                   (int)l.heads, (int)(l.heads / l.qk_heads), (int)l.head_dim, 1, scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool vec = p.dim % 4 == 0 && fits4(pool, l.slot, l.state_head, 0, 16) && fits4(q, l.q_batch, l.q_row, l.q_head, 8) &&
                   fits4(k, l.k_batch, l.k_row, l.k_head, 8);
  if (vec && p.dim % 64 == 0) launch_state_step<DELTA, 2>(p, (int)l.batch, s);
  else if (vec) launch_state_step<DELTA, 1>(p, (int)l.batch, s);
  else launch_state_step<DELTA, 0>(p, (int)l.batch, s);
  return check_launch(what);
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_causal_linear_step(const uint16_t *q, const uint16_t *k, const uint16_t *v, uint16_t *out,
                                        const float *log_decay, float *pool, const int32_t *slots,
                                        const vdnh3_step_layout *layout, float scale, void *stream) {
  return vdnh3::state_step<false>(q, k, v, out, log_decay, nullptr, pool, slots, layout, scale, stream, "causal_linear_step");
}

extern "C" int vdnh3_gated_delta_step(const uint16_t *q, const uint16_t *k, const uint16_t *v, uint16_t *out, const float *beta,
                                      const float *log_decay, float *pool, const int32_t *slots, const vdnh3_step_layout *layout,
                                      void *stream) {
  return vdnh3::state_step<true>(q, k, v, out, log_decay, beta, pool, slots, layout, 1.f, stream, "gated_delta_step");
}
