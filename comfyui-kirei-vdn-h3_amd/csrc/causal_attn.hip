// Causal softmax attention with grouped key / value heads on gfx950, bf16, for the language model that encodes the
// prompts: whole prompts of several sequences packed one behind another, and new tokens over the caches of their
// sequences.
//
//   O_i = sum_{j <= last(i)} p_ij V_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max),  head h reads kv head h / group
//   packed : sequence b is the rows [cu[b], cu[b + 1]) of q, k and v; last(i) = i inside the sequence
//   cached : sequence b has n new tokens in q and the keys 0 .. length[b] - 1 of its cache, the new tokens' last among
//            them; token i sees keys up to length[b] - n + i. One in front of the first key sees none: zeros.
//
// The sequences' bounds are read on the device, so no length is needed on the host and a captured call can be replayed
// with other lengths. Bounds outside the buffers are cut to them.
#include "common.h"

namespace vdnh3 {
namespace {

struct Operand {
  const uint16_t *p;
  int64_t batch, row, head;
  __device__ __forceinline__ const uint16_t *at(int b, int64_t r, int h) const { return p + b * batch + r * row + h * head; }
};

// Where the sequences are: packed (cu set, `batch` strides 0) or cached.
struct Sequences {
  const int32_t *cu, *lengths;
  int count, rows;  // packed: rows of q, k and v; cached: new tokens of a sequence
  int room;         // cached: rows of a cache
};

struct Sequence {
  int q0, n;      // first query row (packed) and number of query rows
  int k0, keys;   // first key row and number of keys
};

__device__ __forceinline__ Sequence sequence_at(const Sequences &s, int b) {
  if (s.cu) {
    const int a = min(max(s.cu[b], 0), s.rows), e = min(max(s.cu[b + 1], a), s.rows);
    return Sequence{a, e - a, a, e - a};
  }
  return Sequence{0, s.rows, 0, min(max(s.lengths[b], 0), s.room)};
}

// The output row of one query by one wavefront: a lane takes a key of each 64, then two (one) channels of the sum.
// Keys that the query does not see are not read.
template <int D>
__device__ __forceinline__ void attend_row(const uint16_t *q, const uint16_t *k, int64_t k_row, const uint16_t *v,
                                           int64_t v_row, int keys, float scale_log2, uint16_t *out, int lane) {
  constexpr int C = D / 64;
  float m = -INFINITY, l = 0.f, o[C] = {};
  for (int j0 = 0; j0 < keys; j0 += 64) {
    float s = -INFINITY;
    if (j0 + lane < keys) {
      const uint16_t *kp = k + (int64_t)(j0 + lane) * k_row;
      float dot = 0.f;
      for (int c = 0; c < D; c += 8) {
        const u32x4_t a = ld16(q + c), b = ld16(kp + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dot = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), dot);
          dot = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(b[i] & 0xffff0000u), dot);
        }
      }
      s = dot * scale_log2;
    }
    const float m_new = fmaxf(m, wave_max(s)), base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = exp2f(m - base), p = exp2f(s - base);  // 0 for a lane without a key
    m = m_new;
    l *= corr;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= corr;
    const int n = min(64, keys - j0);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl(p, j);
      const uint16_t *vp = v + (int64_t)(j0 + j) * v_row + C * lane;
      l += pj;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(pj, bf2f(vp[c]), o[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) out[C * lane + c] = f2bf(keys > 0 ? o[c] / l : 0.f);
}

// One wavefront per (query row, head), four per workgroup.
template <int D>
__global__ __launch_bounds__(256) void causal_rows_kernel(Operand q, Operand k, Operand v, Operand out, Sequences seqs,
                                                          int heads, int group, float scale_log2, int64_t total) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= total) return;
  const int64_t at = w / heads;
  const int head = (int)(w - at * heads), lane = threadIdx.x & 63;
  int b, row;
  if (seqs.cu) {
    row = (int)at;
    int lo = 0, hi = seqs.count;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (seqs.cu[mid] <= row) lo = mid;
      else hi = mid;
    }
    b = lo;
  } else {
    b = (int)(at / seqs.rows);
    row = (int)(at - (int64_t)b * seqs.rows);
  }
  const Sequence s = sequence_at(seqs, b);
  const int i = row - s.q0;
  if (i < 0 || i >= s.n) return;  // no sequence's row
  const int kvh = head / group, keys = min(max(s.keys - s.n + 1 + i, 0), s.keys);
  attend_row<D>(q.at(b, row, head), k.at(b, s.k0, kvh), k.row, v.at(b, s.k0, kvh), v.row, keys, scale_log2,
                const_cast<uint16_t *>(out.at(b, row, head)), lane);
}

int check_operand(const Operand &o, const char *name) {
  VDNH3_HOST_CHECK(o.p != nullptr, VDNH3_ERR_INVALID, "causal attention: %s is null", name);
  VDNH3_HOST_CHECK(o.batch % 8 == 0 && o.row % 8 == 0 && o.head % 8 == 0 && reinterpret_cast<uintptr_t>(o.p) % 16 == 0,
                   VDNH3_ERR_INVALID,
                   "causal attention: %s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  return VDNH3_OK;
}

int check_causal(const Operand &q, const Operand &k, const Operand &v, const Operand &out, int heads, int kv_heads,
                 int head_dim, float scale) {
  VDNH3_HOST_CHECK(head_dim == 64 || head_dim == 128, VDNH3_ERR_INVALID,
                   "causal attention supports head_dim 64 or 128, got %d", head_dim);
  VDNH3_HOST_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, VDNH3_ERR_INVALID,
                   "causal attention: heads (%d) must be a multiple of the key / value heads (%d)", heads, kv_heads);
  VDNH3_HOST_CHECK(scale > 0.f && scale < INFINITY, VDNH3_ERR_INVALID,
                   "causal attention: scale must be positive and finite");
  int rc = check_operand(q, "q");
  if (!rc) rc = check_operand(k, "k");
  if (!rc) rc = check_operand(v, "v");
  if (!rc) rc = check_operand(out, "out");
  return rc;
}

int launch_causal(const Operand &q, const Operand &k, const Operand &v, const Operand &out, const Sequences &seqs,
                  int64_t rows, int heads, int kv_heads, int head_dim, float scale, hipStream_t s) {
  const int64_t total = rows * heads;
  const float scale_log2 = scale * 1.4426950408889634f;
  const int64_t groups = (total + 3) / 4;
  VDNH3_HOST_CHECK(groups <= INT32_MAX, VDNH3_ERR_INVALID, "causal attention: %lld query rows are too many for one launch",
                   (long long)rows);
  const dim3 grid((unsigned)groups);
  if (head_dim == 128)
    hipLaunchKernelGGL(causal_rows_kernel<128>, grid, dim3(256), 0, s, q, k, v, out, seqs, heads, heads / kv_heads,
                       scale_log2, total);
  else
    hipLaunchKernelGGL(causal_rows_kernel<64>, grid, dim3(256), 0, s, q, k, v, out, seqs, heads, heads / kv_heads,
                       scale_log2, total);
  return check_launch("causal attention");
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_causal_attn_packed(const uint16_t *q, int64_t q_row, int64_t q_head, const uint16_t *k, int64_t k_row,
                                        int64_t k_head, const uint16_t *v, int64_t v_row, int64_t v_head, uint16_t *out,
                                        int64_t o_row, int64_t o_head, const int32_t *cu_seqlens, int sequences, int rows,
                                        int heads, int kv_heads, int head_dim, float scale, void *stream) {
  using namespace vdnh3;
  const Operand qo{q, 0, q_row, q_head}, ko{k, 0, k_row, k_head}, vo{v, 0, v_row, v_head}, oo{out, 0, o_row, o_head};
  int rc = check_causal(qo, ko, vo, oo, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  VDNH3_HOST_CHECK(cu_seqlens && sequences > 0 && rows > 0, VDNH3_ERR_INVALID,
                   "causal attention: null sequence bounds, or no sequences or rows");
  return launch_causal(qo, ko, vo, oo, Sequences{cu_seqlens, nullptr, sequences, rows, 0}, rows, heads, kv_heads, head_dim,
                       scale, static_cast<hipStream_t>(stream));
}

extern "C" int vdnh3_causal_attn_cached(const uint16_t *q, int64_t q_batch, int64_t q_row, int64_t q_head,
                                        const uint16_t *k, int64_t k_batch, int64_t k_row, int64_t k_head,
                                        const uint16_t *v, int64_t v_batch, int64_t v_row, int64_t v_head, uint16_t *out,
                                        int64_t o_batch, int64_t o_row, int64_t o_head, const int32_t *lengths, int batch,
                                        int new_tokens, int room, int heads, int kv_heads, int head_dim, float scale,
                                        void *stream) {
  using namespace vdnh3;
  const Operand qo{q, q_batch, q_row, q_head}, ko{k, k_batch, k_row, k_head}, vo{v, v_batch, v_row, v_head},
      oo{out, o_batch, o_row, o_head};
  int rc = check_causal(qo, ko, vo, oo, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  VDNH3_HOST_CHECK(lengths && batch > 0 && new_tokens > 0 && room > 0, VDNH3_ERR_INVALID,
                   "causal attention: null lengths, or no sequences, new tokens or room in the cache");
  return launch_causal(qo, ko, vo, oo, Sequences{nullptr, lengths, batch, new_tokens, room}, (int64_t)batch * new_tokens,
                       heads, kv_heads, head_dim, scale, static_cast<hipStream_t>(stream));
}
