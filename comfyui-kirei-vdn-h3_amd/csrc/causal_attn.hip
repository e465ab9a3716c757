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
#include <algorithm>
#include <cmath>

#include "common.h"
#include "lane_groups.h"

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
// Keys that the query does not see are not read. Probabilities carry a factor of 2^-24, which cancels, so that up to 2^24
// values of bf16's largest sum up inside fp32. An infinite value counts as such also where its key's probability, or what a
// larger score leaves of it, is under fp32's smallest number: the softmax has no zeros but for scores of -inf. L2 bounds it,
// since no two rows share their reads: 2,048 tokens of 40 / 8 heads x 128 that all see an infinite value take 10.7 ms (0.09
// without), 4,096 take 30, but 2,048 take 0.8 where a token is no number, which ends its rows at once.
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
    const float corr = exp2f(m - base), p = exp2f(s - base - 24.f);  // 0 for a lane without a key
    m = m_new;
    l *= corr;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = fabsf(o[c]) == INFINITY ? o[c] : o[c] * corr;
    const int n = min(64, keys - j0);
    const uint64_t faint = __ballot(p == 0.f && s > -INFINITY);
    if (faint == 0) {
      for (int j = 0; j < n; ++j) {
        const float pj = __shfl(p, j);
        const uint16_t *vp = v + (int64_t)(j0 + j) * v_row + C * lane;
        l += pj;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = fmaf(pj, bf2f(vp[c]), o[c]);
      }
    } else {
      for (int j = 0; j < n; ++j) {
        const float pj = __shfl(p, j);
        const uint16_t *vp = v + (int64_t)(j0 + j) * v_row + C * lane;
        l += pj;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float x = bf2f(vp[c]);
          o[c] += ((faint >> j) & 1) && fabsf(x) == INFINITY ? x : pj * x;
        }
      }
    }
    bool number = false;
#pragma unroll
    for (int c = 0; c < C; ++c) number = number || o[c] == o[c];
    if (!(l == l) || !__any(number)) break;  // no channel is a number any more, whatever follows
  }
#pragma unroll
  for (int c = 0; c < C; ++c) out[C * lane + c] = f2bf(keys > 0 ? o[c] / l : 0.f);
}

// ---------------------------------------------------------------------------------
// Whole prompts: one workgroup = 8 wavefronts = 256 rows of one key / value head x the key tiles that they see.
// A row is a (token, query head) pair of the head's group, token-major: row r of a sequence is token r / group and head
// r % group, so every query head of a group shares the workgroup's K and V tiles and a block's rows span few tokens
// (256 rows of 5 heads: 51), which keeps the part of its last tiles that lies behind the diagonal small.
//
// Scores are computed transposed, S^T = K Q^T, on v_mfma_f32_16x16x32_bf16: a lane owns a query of each of its
// wavefront's two 16-query blocks and 24 of a tile's 96 keys, and its probabilities are operands of O^T += V^T P^T as
// they lie. V tiles are loaded as they are, key by key, and read transposed (ds_read_b64_tr_b16: 16 lanes get 4 keys of
// 16 channels), so no pass writes a transposed copy first.
//
// What bounds it: the issue of the SIMD that two wavefronts share. A phase's 102 MFMAs of 16 cycles and the softmax beside
// them, about 1,400 cycles of VALU (a third of it the exponentials), take 2,500 cycles together; LDS is busy for 28% of
// the time, without bank conflicts, and fragment reads 2 to 6 ahead measure the same. 8,296 rows x 40 / 8 heads x 128 take
// 605 us, 1,165 TFLOP/s, where the library's 8,192^3 product reaches 1,367 (585 us on another card). With 64 channels a tile has
// half the products and the same softmax: 8,000 rows x 32 / 8 take 300 us, VALU 55% and matrix cores 39% of them. Short prompts
// are bound by a workgroup's start and end, about 6 us (its block, the first loads, two more phases than tiles, the stores): 512
// rows take 15.1 us.
constexpr int kBN = 96;        // keys per tile
constexpr int kThreads = 512;
constexpr int kRing = 3;       // LDS slots per K and V ring (144 KB at D = 128): loads run kRing - 1 tiles ahead
constexpr int kAhead = 4;      // fragments a wavefront's LDS reads run ahead of its MFMAs
constexpr float kLazy = 8.0f;  // log2 of the largest probability a stale running max allows
constexpr float kNoMax = -3.402823466e38f;  // the running max before any score: finite, so exp2(-inf - max) is 0

// LDS slots: chunk c (16 bytes) of row r lies at slot c ^ swizzle(r). K: the 16 rows of a fragment read hit 16 different
// 16-byte bank groups. V: the 8 rows that half a wavefront reads 32 bytes of hit 8 different 32-byte ones.
template <int D>
__device__ __forceinline__ int k_slot(int r, int c) {
  if constexpr (D == 128) return c ^ (r & 15);
  else return c ^ ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_slot(int r, int c) {
  if constexpr (D == 128) return c ^ (2 * (r & 7));
  else return c ^ (2 * ((r >> 1) & 3));
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));

// Four keys of one channel per lane: 16 lanes read 4 rows of 16 channels (lane i: channels 4 (i % 4) .. + 3 of row i / 4)
// and get their transpose (lane i: channel i of the 4 rows).
__device__ __forceinline__ u32x2_t lds_read_transposed(const uint16_t *p) {
  typedef __attribute__((address_space(3))) s16x4_t *lds_ptr;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p)));
}

// The block of rows a workgroup takes: sequence b, rows [r0, r1) of its n x group.
struct Block {
  int b, r0, r1;
  Sequence s;
};

// Blocks of packed sequences are numbered without a count on the host: sequence b's begin at floor(cu[b] group / BM) + b,
// which leaves room for those before. Every wavefront looks for its own, a lane per sequence and a ballot; of more than 64
// sequences first a 64th (9,000 of one token, 40/8 heads: 1.92 ms, and 6.46 ms with 64 sequences after another looked at).
// Numbers that are no block's give no rows.
template <int BM>
__device__ __forceinline__ Block packed_block(const Sequences &seqs, int block, int group) {
  const int lane = threadIdx.x & 63;
  const Block none{0, 0, 0, Sequence{0, 0, 0, 0}};
  auto from = [&](int b) __device__ { return min(max(seqs.cu[b], 0), seqs.rows); };
  auto begin = [&](int b) __device__ { return (int)((int64_t)from(b) * group / BM) + b; };
  // more than 64: a 64th of them at a time, those of the last that begins at or before the block
  int b0 = 0, count = seqs.count;
  while (count > 64) {
    const int step = (count + 63) / 64, i = lane * step;
    const uint64_t before = __ballot(i < count && begin(b0 + min(i, count - 1)) <= block);
    if (before == 0) return none;
    const int l = 63 - __builtin_clzll(before);
    b0 += l * step;
    count = min(step, count - l * step);
  }
  const int b = b0 + min(lane, count - 1), start = from(b), end = max(from(b + 1), start);
  const uint64_t before = __ballot(lane < count && begin(b) <= block);
  if (before == 0) return none;
  const int l = 63 - __builtin_clzll(before);
  const int a = __builtin_amdgcn_readlane(start, l), n = __builtin_amdgcn_readlane(end, l) - a;
  const int64_t rows = (int64_t)n * group, r0 = (int64_t)(block - __builtin_amdgcn_readlane(begin(b), l)) * BM;
  if (r0 < 0 || r0 >= rows) return none;
  return Block{b0 + l, (int)r0, (int)min(r0 + BM, rows), Sequence{a, n, a, n}};
}

// Caches: every sequence has the same rows.
template <int BM>
__device__ __forceinline__ Block cached_block(const Sequences &seqs, int block, int group) {
  const int rows = seqs.rows * group, per = (rows + BM - 1) / BM, b = block / per, r0 = (block - b * per) * BM;
  return Block{b, r0, min(r0 + BM, rows), sequence_at(seqs, b)};
}

// Two-group ping-pong over the key tiles t = 0 .. T-1: wavefronts 0-3 (group A) and 4-7 (group B) each own 32 rows a
// wavefront; w and w + 4 share a SIMD. In each of the barrier-separated phases p = 0 .. 2T+1 one group works on the matrix
// cores and the other on the VALU:
//   MFMA phase of tile t :  O^T += V(t-1)^T P(t-1)^T, l += 1^T P(t-1)^T, S(t)^T = K(t) Q^T
//   VALU phase of tile t :  P(t) = exp2(scale S(t) - m), row max, O and l rescale
// Group A runs tile t's MFMA phase in phase 2t and its VALU phase in 2t+1; group B one phase later. K(t) and V(t-1) are
// read in phases 2t and 2t+1 only; group A loads K tiles and group B V tiles straight to LDS, each at the start of its VALU
// phase, two tiles ahead. A wavefront leaves out tiles behind its own rows' diagonal.
template <int D, int NQ>
__global__ __launch_bounds__(kThreads, 1) void causal_tile_kernel(Operand q, Operand k, Operand v, Operand out,
                                                                  Sequences seqs, int blocks, int kv_heads, int group,
                                                                  float scale_log2) {
  constexpr int KC = D / 8;      // 16-byte chunks per row
  constexpr int NS = D / 32;     // k-steps of the QK^T contraction
  constexpr int NO = D / 16;     // 16-row blocks of O^T
  constexpr int NKB = kBN / 16;  // 16-key blocks of S^T
  constexpr int NT = kBN / 32;   // k-steps of the PV contraction
  constexpr int TILE = kBN * D;  // elements per tile
  __shared__ __attribute__((aligned(16))) uint16_t Ks[kRing][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t Vs[kRing][TILE];

  // a sequence's last blocks, which see the most keys, first; heads next to each other, so with 8 heads each XCD has its own
  const int kvh = (int)blockIdx.x % kv_heads, block = blocks - 1 - (int)blockIdx.x / kv_heads;
  const Block blk = seqs.cu ? packed_block<128 * NQ>(seqs, block, group) : cached_block<128 * NQ>(seqs, block, group);
  if (blk.r0 >= blk.r1) return;
  const Sequence &sq = blk.s;
  const int behind = sq.keys - sq.n;  // token i sees keys 0 .. behind + i
  const int block_keys = min(behind + (blk.r1 - 1) / group + 1, sq.keys);
  const int T = block_keys > 0 ? (block_keys + kBN - 1) / kBN : 0;

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int l16 = lane & 15, g = lane >> 4;
  const int turn = wave >> 2;  // 0: group A, 1: group B
  const int w0 = blk.r0 + wave * 16 * NQ;  // the wavefront's first row
  const bool rows_live = w0 < blk.r1;
  // the wavefront's tiles, and those of its tiles that need no mask
  const int w_keys = rows_live ? min(behind + (min(w0 + 16 * NQ, blk.r1) - 1) / group + 1, sq.keys) : 0;
  const int w_tiles = __builtin_amdgcn_readfirstlane(w_keys > 0 ? (w_keys + kBN - 1) / kBN : 0);
  const int w_clear = __builtin_amdgcn_readfirstlane(rows_live ? max(behind + w0 / group + 1, 0) / kBN : 0);

  int last[NQ];
  const uint16_t *qp[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = min(w0 + 16 * n + l16, blk.r1 - 1), token = r / group, head = kvh * group + (r - token * group);
    last[n] = behind + token;
    qp[n] = q.at(blk.b, sq.q0 + token, head);
  }

  f32x4_t oacc[NO][NQ], l_run[NQ];
  float m_run[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int m = 0; m < NO; ++m) oacc[m][n] = f32x4_t{};
    m_run[n] = kNoMax;
    l_run[n] = f32x4_t{};
  }

  if (T > 0) {
    // Tile loads, by one group of 256 threads: thread chunk i fills LDS position P = 256 i + gtid (16-byte units): row
    // P / KC, slot P % KC, which holds chunk slot ^ swizzle(row) of that key; the swizzle is the same for every i. Rows
    // past the sequence's keys read its last key (their scores are masked).
    constexpr int CG = kBN * KC / 256;
    const int gtid = tid & 255, kr0 = gtid / KC;
    const int slot = (turn == 0 ? k_slot<D>(kr0, gtid % KC) : v_slot<D>(kr0, gtid % KC)) * 8;
    const int64_t src_row = turn == 0 ? k.row : v.row;
    const uint16_t *src = turn == 0 ? k.at(blk.b, sq.k0, kvh) : v.at(blk.b, sq.k0, kvh);
    uint32_t doff[CG];
#pragma unroll
    for (int i = 0; i < CG; ++i) doff[i] = 2u * ((uint32_t)(kr0 + i * (256 / KC)) * (uint32_t)src_row + slot);
    const uint32_t lds_dma = __builtin_amdgcn_readfirstlane(
        (turn == 0 ? lds_address(&Ks[0][0]) : lds_address(&Vs[0][0])) + (wave & 3) * 64 * 16);
    auto tile_dma = [&](int t, int ring) __device__ {
      const int ks = t * kBN;
      const uint16_t *base = src + (int64_t)ks * src_row;
      uint32_t off[CG];
#pragma unroll
      for (int i = 0; i < CG; ++i) off[i] = doff[i];
      if (ks + kBN > sq.keys) {  // uniform: the last tile only
#pragma unroll
        for (int i = 0; i < CG; ++i)
          off[i] = 2u * ((uint32_t)(min(ks + kr0 + i * (256 / KC), sq.keys - 1) - ks) * (uint32_t)src_row + slot);
      }
#pragma unroll
      for (int i = 0; i < CG; ++i)
        global_to_lds16_sbase(base, off[i], lds_dma + (uint32_t)ring * (TILE * 2) + (uint32_t)(i * 256 * 16));
    };

    // Fragment offsets inside a tile (elements): K by k-step (16-key blocks differ by a constant), V by 16-channel block
    // (its 4-row reads differ by constants: the rows of a lane are 16 a + 4 g + l16 / 4).
    int kfo[NS], vfo[NO];
#pragma unroll
    for (int st = 0; st < NS; ++st) kfo[st] = (l16 * KC + k_slot<D>(l16, 4 * st + g)) * 8;
    const int vr = 4 * g + (l16 >> 2);
#pragma unroll
    for (int m = 0; m < NO; ++m) vfo[m] = vr * D + v_slot<D>(vr, 2 * m + ((l16 >> 1) & 1)) * 8 + 4 * (l16 & 1);

    f32x4_t sacc[NKB][NQ];
    u32x4_t pb[NT][NQ];  // P^T fragments: bf16 pairs
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int n = 0; n < NQ; ++n) pb[j][n] = u32x4_t{};
    const u32x4_t ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};  // eight bf16 1.0

    // K(t) and V(t) live in slot t % kRing. Phase 0 needs K(0), by group A, and the queries; K(1 .. kRing-2) by group A and
    // V(0 .. kRing-3) by group B, which phase 2 needs, follow behind its barrier. V(-1), which the product of tile 0 reads
    // with P(-1) = 0, is zeroed. Group B's first issue in its turn (phase 0) is V(kRing-2).
    if (turn == 0) tile_dma(0, 0);
    bf16x8_t qf[NQ][NS];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[n][s] = as_bf16x8(ld16(qp[n] + 32 * s + 8 * g));
    for (int i = tid; i < TILE / 8; i += kThreads) st16(Vs[kRing - 1] + i * 8, u32x4_t{0, 0, 0, 0});
    wait_vm_lds<0>();
    bare_barrier();
    static_assert(kRing == 3, "one tile of each ring is left to load here");
    if (turn == 0 ? T > 1 : true) tile_dma(turn == 0 ? 1 : 0, turn == 0 ? 1 : 0);

    const int phases = 2 * T + 2;
    for (int p = 0; p < phases; ++p) {
      const int t_mfma = p >> 1, t_valu = (p - 1) >> 1;
      if (turn == (p & 1)) {
        // t = w_tiles has no scores to make and t = 0 no product with values: those halves run on what is there (leaving
        // them out in code of their own carries both operands through the loop, which spills)
        const int t = t_mfma;
        if (t <= w_tiles && w_tiles > 0) {
          const uint16_t *vtile = Vs[(t + kRing - 1) % kRing];
          const uint16_t *ktile = Ks[t % kRing];
          // fragment i < NP: V^T block m = i % NO, k-step i / NO; i >= NP: K block (i - NP) % NKB, k-step (i - NP) / NKB
          constexpr int NP = NO * NT, NF = NP + NKB * NS;
          auto frag = [&](int i) __device__ {
            if (i < NP) {
              const uint16_t *vp = vtile + (i / NO) * 32 * D + vfo[i % NO];
              const u32x2_t a = lds_read_transposed(vp), b = lds_read_transposed(vp + 16 * D);
              return u32x4_t{a[0], a[1], b[0], b[1]};
            }
            return ld16(ktile + ((i - NP) % NKB) * 16 * D + kfo[(i - NP) / NKB]);
          };
          __builtin_amdgcn_s_setprio(1);  // the MFMA wavefront of each SIMD issues ahead of the VALU wavefront beside it
          u32x4_t fr[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) fr[i] = frag(i);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < NF; ++i) {
            const u32x4_t a = fr[i % kAhead];
#pragma unroll
            for (int x = 0; x < NQ; ++x) {
              const int n = (i & 1) ? NQ - 1 - x : x;
              if (i < NP) {
                oacc[i % NO][n] = mfma_bf16_16x16x32(as_bf16x8(a), as_bf16x8(pb[i / NO][n]), oacc[i % NO][n]);
                if (i % NO == NO - 1)
                  l_run[n] = mfma_bf16_16x16x32(as_bf16x8(ones), as_bf16x8(pb[i / NO][n]), l_run[n]);
              } else {
                const int kb = (i - NP) % NKB, st = (i - NP) / NKB;
                if (st == 0) sacc[kb][n] = f32x4_t{};
                sacc[kb][n] = mfma_bf16_16x16x32(as_bf16x8(a), qf[n][st], sacc[kb][n]);
              }
            }
            if (i + kAhead < NF) fr[i % kAhead] = frag(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(0);
        }
      } else {
        if (t_valu + kRing - 1 < T) tile_dma(t_valu + kRing - 1, (t_valu + kRing - 1) % kRing);
        if (p >= 1 + turn && t_valu < w_tiles) {
          if (t_valu >= w_clear) {  // part of the tile lies behind a row
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              const int seen = last[n] - t_valu * kBN - 4 * g;
#pragma unroll
              for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) sacc[kb][n][i] = 16 * kb + i > seen ? -INFINITY : sacc[kb][n][i];
            }
          }
          static_assert(NKB == 6 && NQ <= 2, "the max tree is written for 24 scores per lane and query");
          float mt[NQ];
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float m1[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              m1[i] = fmaxf(fmaxf(sacc[0][n][i], sacc[1][n][i]), sacc[2][n][i]);
              m1[4 + i] = fmaxf(fmaxf(sacc[3][n][i], sacc[4][n][i]), sacc[5][n][i]);
            }
            const float a = fmaxf(fmaxf(m1[0], m1[1]), m1[2]), b = fmaxf(fmaxf(m1[3], m1[4]), m1[5]);
            mt[n] = fmaxf(fmaxf(a, b), fmaxf(m1[6], m1[7]));
          }
          group_max(mt[0], mt[NQ - 1]);
          bool grow = false;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mt[n] *= scale_log2;
            grow = grow || mt[n] > m_run[n] + kLazy;
          }
          if (__any(grow)) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              const float m_new = mt[n] > m_run[n] + kLazy ? mt[n] : m_run[n];
              const float corr = __builtin_amdgcn_exp2f(m_run[n] - m_new);
              m_run[n] = m_new;
              l_run[n] *= corr;
#pragma unroll
              for (int m = 0; m < NO; ++m) oacc[m][n] *= corr;
            }
          }
          // P in bf16 pairs, the matrix cores' operand, for the PV product and the row sums alike: up to 2^-8 of a
          // probability, 2.0e-3 of the result in 2-norm with its own rounding's 1.6e-3
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sacc[kb][n][i], scale_log2, -m_run[n]));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sacc[kb][n][i + 1], scale_log2, -m_run[n]));
                pb[kb >> 1][n][2 * (kb & 1) + (i >> 1)] = pack_bf2(p0, p1);
              }
        }
      }
      // before an even phase 2(t+1): K(t+1) and V(t) have landed. While there are tiles to load, each group's latest one,
      // K(t+2) or V(t+1), may still be in flight; after that there is none later.
      if (p & 1) {
        if (t_valu + kRing - 1 < T) wait_vm_lds<(kRing - 2) * CG>();
        else wait_vm_lds<0>();
      }
      bare_barrier();
    }
  }

  // The rows leave through LDS, whole: a lane holds 4 channels of 16 blocks each, and stores of 8 bytes to 16 rows take
  // longer than this. Row r's 16-byte chunk c lies at chunk c ^ (r % 16) of its wavefront's part of the K ring.
  uint16_t *mine = &Ks[0][0] + wave * (16 * NQ * D);
  bool again[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float inv = last[n] >= 0 ? 1.f / l_run[n][0] : 0.f;  // a row that sees nothing gives zeros
    float odd = 0.f;  // 0 as long as every value is finite, then a NaN
#pragma unroll
    for (int m = 0; m < NO; ++m) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = oacc[m][n][i] * inv;
        odd = fmaf(o[i], 0.f, odd);
      }
      *reinterpret_cast<uint2 *>(mine + (16 * n + l16) * D + (((2 * m + (g >> 1)) ^ l16) & (KC - 1)) * 8 + 4 * (g & 1)) =
          make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
    }
    again[n] = !(odd == 0.f) && w0 + 16 * n + l16 < blk.r1;
  }
  {
    constexpr int RPI = 64 / KC;  // rows per instruction
    const int c = lane % KC;
    int r = lane / KC, token = (w0 + r) / group, head = w0 + r - token * group;
    const int tokens = RPI / group, heads = RPI - tokens * group;
#pragma unroll
    for (int i = 0; i < 16 * NQ / RPI; ++i) {
      if (w0 + r < blk.r1)
        st16(const_cast<uint16_t *>(out.at(blk.b, sq.q0 + token, kvh * group + head)) + 8 * c,
             ld16(mine + r * D + ((c ^ r) & (KC - 1)) * 8));
      r += RPI;
      token += tokens;
      head += heads;
      if (head >= group) {
        head -= group;
        ++token;
      }
    }
  }
  // A value that is not finite behind a row, in a tile that the row sees a part of, times the row's probability 0 is a NaN
  // in its sum. Rows whose result is not finite are computed once more without the keys that they do not see: never for
  // finite inputs whose result bf16 holds.
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    uint64_t todo = __ballot(again[n]);
    todo |= todo >> 32;
    todo |= todo >> 16;
    if (todo) wait_vm_lds<0>();  // the stores above come first
    for (uint32_t rows = (uint32_t)todo & 0xffffu; rows; rows &= rows - 1) {
      const int r = w0 + 16 * n + __builtin_ctz(rows), token = r / group, head = kvh * group + (r - token * group);
      attend_row<D>(q.at(blk.b, sq.q0 + token, head), k.at(blk.b, sq.k0, kvh), k.row, v.at(blk.b, sq.k0, kvh), v.row,
                    min(behind + token + 1, sq.keys), scale_log2, const_cast<uint16_t *>(out.at(blk.b, sq.q0 + token, head)),
                    lane);
    }
  }
}

// ---------------------------------------------------------------------------------
// Few rows over long caches (new tokens): what counts is to stream the keys and values once. The 32-key tiles of all
// sequences, one behind another, are cut into `ranges` equal ranges for each key / value head, one workgroup each and mostly
// one workgroup per CU: whatever the lengths are, every CU streams the same number of tiles, in one round. A range crosses
// from one sequence into the next; only the sequences at its two ends can be shared with other ranges. Such a part is
// written unnormalised in fp32 with its max and sum and combined by a second launch; a sequence inside a range is finished at
// once. The cut follows from the lengths on the device, in both kernels alike.
//
// A workgroup takes 16 NQ of a head's (token, head) rows, up to 48 (64 spill). Its wavefronts take the tiles in turn, each
// through two LDS slots of its own (one tile in flight while it works on the other, no barrier), with a running softmax of its
// own; they are merged in LDS at the end of a sequence. HBM bounds it: 64 requests of up to 8,192 keys x 8 heads x 128
// (1.1 GB) take 196 us, 5.6 TB/s where a copy reaches 4.8; one request of 40,688 keys (167 MB) 30 us and 6 for the
// combination, which is a launch and a chain of three loads. 32 new tokens over them (four blocks of rows, 78 MFMAs a tile) take
// 91 us: a chain too, of a tile's products, maxima and exponentials in the only wavefront of a SIMD. With fixed chunks of keys
// instead of equal ranges the 64 requests took 215 to 244 us, whole rounds of workgroups each with a pipeline to fill.
constexpr int kFewKeys = 32;      // keys per tile: one k-step of the PV product
constexpr int kFewRing = 2;
// Tiles of a range, at least: one per wavefront (one request of 1,000 keys x 40 / 8 heads: 16 ranges 11.1 us, 8 11.3, 4
// 12.2).
constexpr int kFewLeast = 4;
constexpr int kFewThreads = 256;  // of both kernels

// Unnormalised results of the ranges' ends: [kv head][range][end][row] of D floats, then the same of (max, sum).
struct Parts {
  float *o;
  float2 *ml;
  int ranges;
  __device__ __forceinline__ int64_t at(int kvh, int range, int end, int rows) const {
    return (((int64_t)kvh * ranges + range) * 2 + end) * rows;
  }
};

__device__ __forceinline__ int keys_of(const Sequences &seqs, int b) { return min(max(seqs.lengths[b], 0), seqs.room); }
// The tiles of a sequence; one without keys has one, which writes its rows.
__device__ __forceinline__ int tiles_of(int keys) { return max(1, (keys + kFewKeys - 1) / kFewKeys); }
__device__ __forceinline__ int tiles_of(const Sequences &seqs, int b) { return tiles_of(keys_of(seqs, b)); }

// How the tiles of all sequences are cut: `each` per range, the first `more` ranges one more. Each of the workgroup's
// threads counts the tiles of `per` sequences; before[i] is what the threads in front of i counted.
struct Cut {
  int total, per, ranges, each, more;
  const int *before;
  __device__ __forceinline__ int start(int range) const { return range * each + min(range, more); }
  __device__ __forceinline__ int range_of(int u) const {
    return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each;
  }
  // tiles in front of sequence b
  __device__ __forceinline__ int in_front(const Sequences &seqs, int b) const {
    int u = before[b / per];
    for (int i = b / per * per; i < b; ++i) u += tiles_of(seqs, i);
    return u;
  }
};
__device__ __forceinline__ Cut make_cut(const Sequences &seqs, int ranges, int (&before)[kFewThreads]) {
  __shared__ int waves[kFewThreads / 64];
  const int tid = threadIdx.x, per = (seqs.count + kFewThreads - 1) / kFewThreads;
  int own = 0;
  for (int b = tid * per; b < min((tid + 1) * per, seqs.count); ++b) own += tiles_of(seqs, b);
  int sum = own;  // up to and with this lane's
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(sum, o);
    if ((tid & 63) >= o) sum += x;
  }
  if ((tid & 63) == 63) waves[tid >> 6] = sum;
  __syncthreads();
  int front = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kFewThreads / 64; ++w) {
    if (w < tid >> 6) front += waves[w];
    total += waves[w];
  }
  before[tid] = front + sum - own;
  __syncthreads();
  const int n = min(ranges, max(total / kFewLeast, 1)), each = total / n;
  return Cut{total, per, n, each, total - n * each, before};
}

// A row of the result by `attend_row`. A value that is not finite gives a NaN where it meets a probability of 0: that of a key
// behind the row, of a last key that stands in for one, or what the rounding of its own probability left. Values near
// fp32's largest can sum up past it. Rows with such a result are computed once more, from the keys that they see.
template <int D>
__device__ __forceinline__ void again_row(const Operand &q, const Operand &k, const Operand &v, const Operand &out,
                                          const Sequence &s, int b, int kvh, int group, int row, float scale_log2, int lane) {
  const int token = row / group, head = kvh * group + (row - token * group);
  attend_row<D>(q.at(b, s.q0 + token, head), k.at(b, s.k0, kvh), k.row, v.at(b, s.k0, kvh), v.row,
                min(s.keys - s.n + token + 1, s.keys), scale_log2, const_cast<uint16_t *>(out.at(b, s.q0 + token, head)), lane);
}

template <int D, int NQ>
__global__ __launch_bounds__(kFewThreads) void causal_few_kernel(Operand q, Operand k, Operand v, Operand out, Sequences seqs,
                                                                 int kv_heads, int group, int row_blocks, float scale_log2,
                                                                 Parts parts) {
  constexpr int KC = D / 8, NS = D / 32, NO = D / 16, ROWS = 16 * NQ, W = kFewThreads / 64;
  constexpr int TILE = kFewKeys * D;  // elements
  static_assert(ROWS * D * 2 <= kFewRing * 2 * TILE, "a wavefront's sums fit its tiles' place");
  __shared__ __attribute__((aligned(16))) uint16_t tiles[W][kFewRing][2][TILE];
  __shared__ float2 stats[W][ROWS];
  __shared__ int before[kFewThreads];

  // heads next to each other, whose rows lie side by side in a cache, then the row blocks, which read the same keys
  const int kvh = (int)blockIdx.x % kv_heads, rb = (int)blockIdx.x / kv_heads % row_blocks;
  const int range = (int)blockIdx.x / (kv_heads * row_blocks);
  const Cut cut = make_cut(seqs, parts.ranges, before);
  if (range >= cut.ranges) return;
  int u = cut.start(range);
  const int u1 = cut.start(range + 1);
  const int rows = seqs.rows * group, r0 = rb * ROWS, r1 = min(r0 + ROWS, rows);

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int l16 = lane & 15, g = lane >> 4;
  // the sequence that holds tile u, and the tiles in front of it
  int b = 0;
  {
    int lo = 0, hi = kFewThreads;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= u) lo = mid;
      else hi = mid;
    }
    b = lo * cut.per;
  }
  int front = before[b / cut.per];
  int keys = keys_of(seqs, b), here = tiles_of(keys);
  while (front + here <= u) {
    front += here;
    keys = keys_of(seqs, ++b);
    here = tiles_of(keys);
  }
  for (bool first_part = true; u < u1; first_part = false) {
    const Sequence s{0, seqs.rows, 0, keys};
    const int next_keys = keys_of(seqs, min(b + 1, seqs.count - 1));  // on its way while this one is worked on
    const int behind = s.keys - s.n;
    const int k0 = (u - front) * kFewKeys;
    const int n_units = min(u1, front + here) - u;
    const int k1 = min(k0 + n_units * kFewKeys, s.keys);
    const int n_tiles = s.keys > 0 ? n_units : 0;
    const int clear = behind + r0 / group + 1;  // every row sees keys below it
    bf16x8_t qf[NQ][NS];
    int last[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = min(r0 + 16 * n + l16, r1 - 1), token = r / group, head = kvh * group + (r - token * group);
      last[n] = behind + token;
      const uint16_t *qp = q.at(b, s.q0 + token, head) + 8 * g;
#pragma unroll
      for (int st = 0; st < NS; ++st) qf[n][st] = as_bf16x8(ld16(qp + 32 * st));
    }

    // A wavefront's load of a tile: instruction i brings rows i * 64 / KC + lane / KC, slot lane % KC (swizzled as in the
    // kernel above). Rows past the part's keys read its last one (their scores are masked).
    constexpr int LOADS = kFewKeys * KC / 64;
    const int lr = lane / KC;
    const uint16_t *kb = k.at(b, s.k0, kvh), *vb = v.at(b, s.k0, kvh);
    const uint32_t lds0 = lds_address(&tiles[wave][0][0][0]);
    auto load_tile = [&](int t, int ring) __device__ {
      const int key = k0 + t * kFewKeys;
      const uint16_t *kt = kb + (int64_t)key * k.row, *vt = vb + (int64_t)key * v.row;
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int r = i * (64 / KC) + lr;
          const int slot = which ? v_slot<D>(r, lane % KC) : k_slot<D>(r, lane % KC);
          const uint32_t row = (uint32_t)(min(key + r, k1 - 1) - key);
          global_to_lds16_sbase(which ? vt : kt, 2u * (row * (uint32_t)(which ? v.row : k.row) + slot * 8),
                                lds0 + (uint32_t)((ring * 2 + which) * TILE * 2 + i * 1024));
        }
    };
    int kfo[NS], vfo[NO];
#pragma unroll
    for (int st = 0; st < NS; ++st) kfo[st] = (l16 * KC + k_slot<D>(l16, 4 * st + g)) * 8;
    const int vr = 4 * g + (l16 >> 2);
#pragma unroll
    for (int m = 0; m < NO; ++m) vfo[m] = vr * D + v_slot<D>(vr, 2 * m + ((l16 >> 1) & 1)) * 8 + 4 * (l16 & 1);

    f32x4_t oacc[NO][NQ], l_run[NQ];
    float m_run[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int m = 0; m < NO; ++m) oacc[m][n] = f32x4_t{};
      m_run[n] = kNoMax;
      l_run[n] = f32x4_t{};
    }
    const u32x4_t ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};  // eight bf16 1.0

    if (wave < n_tiles) load_tile(wave, 0);
    if (wave + W < n_tiles) load_tile(wave + W, 1);
    // The queries arrive here: the compiler counts its own loads only, so that its wait for them, in the loop, would be one
    // for every tile on its way.
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        u32x4_t x = __builtin_bit_cast(u32x4_t, qf[n][st]);
        asm volatile("" : "+v"(x));
        qf[n][st] = as_bf16x8(x);
      }
    int ring = 0;
    for (int t = wave; t < n_tiles; t += W, ring ^= 1) {
      if (t + W < n_tiles) wait_vm_lds<2 * LOADS>();
      else wait_vm_lds<0>();
      asm volatile("" ::: "memory");
      const uint16_t *ktile = tiles[wave][ring][0], *vtile = tiles[wave][ring][1];
      f32x4_t sacc[2][NQ];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) sacc[h][n] = f32x4_t{};
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const bf16x8_t a = as_bf16x8(ld16(ktile + h * 16 * D + kfo[st]));
#pragma unroll
          for (int n = 0; n < NQ; ++n) sacc[h][n] = mfma_bf16_16x16x32(a, qf[n][st], sacc[h][n]);
        }
      }
      const int key = k0 + t * kFewKeys;
      if (key + kFewKeys > min(clear, k1)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at_key = key + 16 * h + 4 * g + i;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              if (at_key > last[n] || at_key >= k1) sacc[h][n][i] = -INFINITY;
          }
      }
      // P as bf16 and what that leaves, again as bf16 (16 bits of each probability): the matrix cores are idle beside the
      // loads, and the result is then as exact as its own rounding
      u32x4_t pb[NQ], pl[NQ];
      float mt[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const f32x4_t x = sacc[0][n], y = sacc[1][n];
        mt[n] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
      }
#pragma unroll
      for (int n = 0; n < NQ; n += 2) group_max(mt[n], mt[min(n + 1, NQ - 1)]);
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        mt[n] *= scale_log2;
        grow = grow || mt[n] > m_run[n] + kLazy;
      }
      if (__any(grow)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float m_new = mt[n] > m_run[n] + kLazy ? mt[n] : m_run[n];
          const float corr = __builtin_amdgcn_exp2f(m_run[n] - m_new);
          m_run[n] = m_new;
          l_run[n] *= corr;
#pragma unroll
          for (int m = 0; m < NO; ++m) oacc[m][n] *= corr;
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(sacc[h][n][i], scale_log2, -m_run[n]));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(sacc[h][n][i + 1], scale_log2, -m_run[n]));
            const uint32_t w = pack_bf2(p0, p1);
            pb[n][2 * h + (i >> 1)] = w;
            pl[n][2 * h + (i >> 1)] = pack_bf2(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
          }
        l_run[n] = mfma_bf16_16x16x32(as_bf16x8(ones), as_bf16x8(pb[n]), l_run[n]);
        l_run[n] = mfma_bf16_16x16x32(as_bf16x8(ones), as_bf16x8(pl[n]), l_run[n]);
      }
#pragma unroll
      for (int m = 0; m < NO; ++m) {
        const u32x2_t x = lds_read_transposed(vtile + vfo[m]), y = lds_read_transposed(vtile + 16 * D + vfo[m]);
        const bf16x8_t a = as_bf16x8(u32x4_t{x[0], x[1], y[0], y[1]});
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          oacc[m][n] = mfma_bf16_16x16x32(a, as_bf16x8(pb[n]), oacc[m][n]);
          oacc[m][n] = mfma_bf16_16x16x32(a, as_bf16x8(pl[n]), oacc[m][n]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this tile is read: the one after the next comes over it
      if (t + 2 * W < n_tiles) load_tile(t + 2 * W, ring);
    }

    // Each wavefront's sums into its tiles' place: row 16 n + l16, 16-byte chunk 4 m + g at chunk ^ (row % 16).
    float *mine = reinterpret_cast<float *>(&tiles[wave][0][0][0]);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = 16 * n + l16;
#pragma unroll
      for (int m = 0; m < NO; ++m)
        *reinterpret_cast<f32x4_t *>(mine + r * D + 4 * ((4 * m + g) ^ l16)) = oacc[m][n];
      if (g == 0) stats[wave][r] = make_float2(m_run[n], l_run[n][0]);
    }
    __syncthreads();
    constexpr int LANES = D / 4, AT_ONCE = kFewThreads / LANES;  // of a row, four channels each; rows at once
    for (int first_row = 0; first_row < r1 - r0; first_row += AT_ONCE) {
      const int r = min(first_row + tid / LANES, r1 - r0 - 1), c = tid % LANES;
      const bool live = first_row + tid / LANES < r1 - r0;
      float top = kNoMax, l = 0.f;
      float2 ml[W];
      f32x4_t o = {};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        ml[w] = stats[w][r];
        top = fmaxf(top, ml[w].x);
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float by = __builtin_amdgcn_exp2f(ml[w].x - top);
        l = fmaf(by, ml[w].y, l);
        o += by * *reinterpret_cast<const f32x4_t *>(reinterpret_cast<const float *>(&tiles[w][0][0][0]) + r * D + 4 * (c ^ (r & 15)));
      }
      if (n_units == here) {
        const int token = (r0 + r) / group, head = kvh * group + (r0 + r - token * group);
        const float inv = behind + token >= 0 && s.keys > 0 ? 1.f / l : 0.f;
        o *= inv;
        const bool odd = live && !(fmaf(o[0], 0.f, fmaf(o[1], 0.f, fmaf(o[2], 0.f, o[3] * 0.f))) == 0.f);
        if (live)
          *reinterpret_cast<uint2 *>(const_cast<uint16_t *>(out.at(b, s.q0 + token, head)) + 4 * c) =
              make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
        const uint64_t odds = __ballot(odd);
        if (odds) {
          wait_vm_lds<0>();  // the stores above come first
          for (int i = 0; i < 64 / LANES; ++i)
            if ((odds >> (i * LANES)) & ((1ull << LANES) - 1))
              again_row<D>(q, k, v, out, s, b, kvh, group, r0 + first_row + wave * (64 / LANES) + i, scale_log2, lane);
        }
      } else if (live) {
        const int64_t to = parts.at(kvh, range, first_part ? 0 : 1, rows) + r0 + r;
        *reinterpret_cast<f32x4_t *>(parts.o + to * D + 4 * c) = o;
        if (c == 0) parts.ml[to] = make_float2(top, l);
      }
    }
    u += n_units;
    if (u < u1) {
      front += here;
      ++b;
      keys = next_keys;
      here = tiles_of(keys);
      __syncthreads();  // the sums are read: the next sequence's tiles load over them
    }
  }
}

// The rows of sequences that several ranges share, `per` rows of one sequence and key / value head per workgroup: of few
// parts a row per wavefront, of many all wavefronts on one row, merged in LDS. A wavefront has eight parts on their way at
// once (its loads do not wait for one another's maxima).
template <int D>
__global__ __launch_bounds__(kFewThreads) void causal_combine_kernel(Operand q, Operand k, Operand v, Operand out,
                                                                     Sequences seqs, int kv_heads, int group, int per,
                                                                     float scale_log2, Parts parts) {
  constexpr int C = D / 64, W = kFewThreads / 64, AT_ONCE = 8;
  __shared__ float sums[W][D];
  __shared__ float2 stats[W];
  __shared__ int before[kFewThreads];
  const int rows = seqs.rows * group, row_blocks = (rows + per - 1) / per;
  const int bh = (int)blockIdx.x / row_blocks, row0 = ((int)blockIdx.x - bh * row_blocks) * per, b = bh / kv_heads;
  const int kvh = bh - b * kv_heads, row1 = min(row0 + per, rows);
  const Cut cut = make_cut(seqs, parts.ranges, before);
  const int u = cut.in_front(seqs, b);
  const int first = cut.range_of(u), past = cut.range_of(u + tiles_of(seqs, b) - 1) + 1;
  if (past - first == 1) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // a range's part of the sequence is its first one, but in a range that began in an earlier sequence
  const int early = cut.start(first) < u ? first : -1;
  const Sequence s = sequence_at(seqs, b);
  // parts begin, begin + step, ... of a row: their sum, weight and max
  auto gather = [&](int row, int begin, int step, float (&o)[C], float &l, float &m) __device__ {
    m = kNoMax;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
    for (int i0 = begin; i0 < past; i0 += step * AT_ONCE) {
      float2 ml[AT_ONCE];
      float x[AT_ONCE][C];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int i = min(i0 + step * j, past - 1);
        const int64_t from = parts.at(kvh, i, i == early, rows) + row;
        ml[j] = parts.ml[from];
#pragma unroll
        for (int c = 0; c < C; ++c) x[j][c] = parts.o[from * D + C * lane + c];
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (i0 + step * j < past) top = fmaxf(top, ml[j].x);
      const float by = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= by;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= by;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (i0 + step * j >= past) break;
        const float f = __builtin_amdgcn_exp2f(ml[j].x - top);
        l = fmaf(f, ml[j].y, l);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = fmaf(f, x[j][c], o[c]);
      }
    }
  };
  auto finish = [&](int row, float (&o)[C], float l) __device__ {
    const int token = row / group, head = kvh * group + (row - token * group);
    const float inv = s.keys - s.n + token >= 0 ? 1.f / l : 0.f;
    float odd = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      o[c] *= inv;
      odd = fmaf(o[c], 0.f, odd);
    }
    if (__any(!(odd == 0.f))) {
      again_row<D>(q, k, v, out, s, b, kvh, group, row, scale_log2, lane);
      return;
    }
    uint16_t *op = const_cast<uint16_t *>(out.at(b, s.q0 + token, head));
    if constexpr (C == 2) *reinterpret_cast<uint32_t *>(op + 2 * lane) = pack_bf2(o[0], o[1]);
    else op[lane] = f2bf(o[0]);
  };
  float o[C], l, m;
  if (past - first <= AT_ONCE && per >= W) {
    for (int row = row0 + wave; row < row1; row += W) {
      gather(row, first, 1, o, l, m);
      finish(row, o, l);
    }
    return;
  }
  for (int row = row0; row < row1; ++row) {
    gather(row, first + wave, W, o, l, m);
    if (row > row0) __syncthreads();  // the last row's sums are read
#pragma unroll
    for (int c = 0; c < C; ++c) sums[wave][C * lane + c] = o[c];
    if (lane == 0) stats[wave] = make_float2(m, l);
    __syncthreads();
    if (wave) continue;
    float top = kNoMax;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w].x);
    l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float by = __builtin_amdgcn_exp2f(stats[w].x - top);
      l = fmaf(by, stats[w].y, l);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(by, sums[w][C * lane + c], o[c]);
    }
    finish(row, o, l);
  }
}

constexpr float kLog2E = 1.4426950408889634f;

// Rows of a cache: keys are counted in 32 bits, up to the end of a tile behind the last.
constexpr int kMostRoom = INT32_MAX - 4 * kBN;

// A dimension of one element has no stride, whatever a caller passes for it.
Operand operand(const uint16_t *p, int64_t batch, int64_t row, int64_t head, int batches, int rows, int heads) {
  return Operand{p, batches > 1 ? batch : 0, rows > 1 ? row : 0, heads > 1 ? head : 0};
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
  VDNH3_HOST_CHECK(scale > 0.f && scale * kLog2E < INFINITY, VDNH3_ERR_INVALID,
                   "causal attention: scale must be positive, and finite times log2(e)");
  int rc = check_operand(q, "q");
  if (!rc) rc = check_operand(k, "k");
  if (!rc) rc = check_operand(v, "v");
  if (!rc) rc = check_operand(out, "out");
  if (rc) return rc;
  // a lane's offset inside a tile, 95 rows and a row's channels, stays under 2^31 bytes
  VDNH3_HOST_CHECK(k.row >= 0 && v.row >= 0 && k.row <= (1 << 23) && v.row <= (1 << 23), VDNH3_ERR_INVALID,
                   "causal attention: rows of k and v may be at most %d elements apart", 1 << 23);
  return VDNH3_OK;
}

template <int D, int NQ>
int launch_tiles(const Operand &q, const Operand &k, const Operand &v, const Operand &out, const Sequences &seqs, int heads,
                 int kv_heads, float scale, hipStream_t s) {
  constexpr int BM = 128 * NQ;
  const int group = heads / kv_heads;
  VDNH3_HOST_CHECK((int64_t)seqs.rows * group <= INT32_MAX - BM, VDNH3_ERR_INVALID,
                   "causal attention: %d rows of %d heads are too many", seqs.rows, heads);
  const int64_t blocks = seqs.cu ? (int64_t)seqs.rows * group / BM + seqs.count
                                 : seqs.count * (((int64_t)seqs.rows * group + BM - 1) / BM);
  int rc = check_grid(blocks, kThreads, "causal attention");
  if (!rc) rc = check_grid(blocks * kv_heads, kThreads, "causal attention");
  if (rc) return rc;
  hipLaunchKernelGGL((causal_tile_kernel<D, NQ>), dim3((unsigned)(blocks * kv_heads)), dim3(kThreads), 0, s, q, k, v, out, seqs,
                     (int)blocks, kv_heads, group, scale * kLog2E);
  return check_launch("causal attention");
}

// Workgroups of 256 rows from which on they are taken; with fewer, workgroups of 128 (which read twice the LDS for the same
// products) leave fewer CUs without one and end closer together. 512 rows x 40 / 8 x 128 15 us against 23, 4,148 x 16 / 2
// (260 workgroups) 88 against 98, 2,000 x 40 / 8 (313) 67 against 60, 8,296 751 against 588; with 64 channels, where two of 128
// rows fit a CU (125 registers; 256 rows take 186, one workgroup), 4,000 x 20 / 20 (313) 65 against 74, 8,000 x 32 / 8 (1,000)
// 325 against 296.
constexpr int kHighGroups128 = 288, kHighGroups64 = 512;

bool high_blocks(int sequences, int rows, int heads, int head_dim) {
  return (double)rows * sequences * heads / 256 >= (head_dim == 128 ? kHighGroups128 : kHighGroups64);
}

int launch_causal(const Operand &q, const Operand &k, const Operand &v, const Operand &out, const Sequences &seqs, int heads,
                  int kv_heads, int head_dim, float scale, hipStream_t s) {
  const bool high = high_blocks(seqs.cu ? 1 : seqs.count, seqs.rows, heads, head_dim);
  if (head_dim == 128)
    return high ? launch_tiles<128, 2>(q, k, v, out, seqs, heads, kv_heads, scale, s)
                : launch_tiles<128, 1>(q, k, v, out, seqs, heads, kv_heads, scale, s);
  return high ? launch_tiles<64, 2>(q, k, v, out, seqs, heads, kv_heads, scale, s)
              : launch_tiles<64, 1>(q, k, v, out, seqs, heads, kv_heads, scale, s);
}

// Rows of a workgroup: equal blocks of up to 48, in 16s.
int few_block(int64_t rows) {
  const int64_t blocks = (rows + 47) / 48;
  return (int)((rows + 16 * blocks - 1) / (16 * blocks)) * 16;
}

template <int D, int NQ>
int launch_few(const Operand &q, const Operand &k, const Operand &v, const Operand &out, const Sequences &seqs, int kv_heads,
               int group, float scale_log2, const Parts &parts, hipStream_t s) {
  const int rows = seqs.rows * group, row_blocks = (rows + 16 * NQ - 1) / (16 * NQ);
  const int64_t blocks = (int64_t)kv_heads * row_blocks * parts.ranges;
  int rc = check_grid(blocks, kFewThreads, "causal attention over caches");
  // a row per workgroup up to four workgroups a CU, then fours of rows: every workgroup has the cut to make first
  const int64_t all = (int64_t)seqs.count * kv_heads * rows;
  const int per = all <= 1024 ? 1 : (int)std::min<int64_t>((all + 4095) / 4096 * 4, rows);
  const int64_t combines = (int64_t)seqs.count * kv_heads * ((rows + per - 1) / per);
  if (!rc) rc = check_grid(combines, kFewThreads, "causal attention over caches");
  if (rc) return rc;
  hipLaunchKernelGGL((causal_few_kernel<D, NQ>), dim3((unsigned)blocks), dim3(kFewThreads), 0, s, q, k, v, out, seqs, kv_heads,
                     group, row_blocks, scale_log2, parts);
  rc = check_launch("causal attention over caches");
  if (rc || parts.ranges == 1) return rc;
  hipLaunchKernelGGL(causal_combine_kernel<D>, dim3((unsigned)combines), dim3(kFewThreads), 0, s, q, k, v, out, seqs,
                     kv_heads, group, per, scale_log2, parts);
  return check_launch("causal attention's ranges");
}

template <int D>
int launch_few_rows(const Operand &q, const Operand &k, const Operand &v, const Operand &out, const Sequences &seqs,
                    int kv_heads, int group, float scale_log2, const Parts &parts, hipStream_t s) {
  switch (few_block((int64_t)seqs.rows * group)) {
    case 16: return launch_few<D, 1>(q, k, v, out, seqs, kv_heads, group, scale_log2, parts, s);
    case 32: return launch_few<D, 2>(q, k, v, out, seqs, kv_heads, group, scale_log2, parts, s);
    default: return launch_few<D, 3>(q, k, v, out, seqs, kv_heads, group, scale_log2, parts, s);
  }
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_causal_attn_packed(const uint16_t *q, int64_t q_row, int64_t q_head, const uint16_t *k, int64_t k_row,
                                        int64_t k_head, const uint16_t *v, int64_t v_row, int64_t v_head, uint16_t *out,
                                        int64_t o_row, int64_t o_head, const int32_t *cu_seqlens, int sequences, int rows,
                                        int heads, int kv_heads, int head_dim, float scale, void *stream) {
  using namespace vdnh3;
  const Operand qo = operand(q, 0, q_row, q_head, 1, rows, heads), ko = operand(k, 0, k_row, k_head, 1, rows, kv_heads),
                vo = operand(v, 0, v_row, v_head, 1, rows, kv_heads), oo = operand(out, 0, o_row, o_head, 1, rows, heads);
  int rc = check_causal(qo, ko, vo, oo, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  VDNH3_HOST_CHECK(cu_seqlens && sequences > 0 && rows > 0, VDNH3_ERR_INVALID,
                   "causal attention: null sequence bounds, or no sequences or rows");
  return launch_causal(qo, ko, vo, oo, Sequences{cu_seqlens, nullptr, sequences, rows, 0}, heads, kv_heads, head_dim, scale,
                       static_cast<hipStream_t>(stream));
}

// The ranges of a call, or 0 for the kernel above: whichever an estimate says takes the least time, in us. The lengths are not
// known here: caches are taken to be 64% full, the longest whole.
//   0      : 4 + the longer of the bytes at 7.5 TB/s (partly out of the last-level cache) and 0.9 (64 channels: 0.75) per 96
//            keys of the longest cache and round of workgroups (128 rows of one sequence and key / value head each)
//   ranges : 10 (of more than 16 rows a workgroup: 13), 5.3 less for a single range, which needs no combination, + 0.08 per
//            range of a sequence + 4.2 per further round of workgroups + the longer of the bytes at 8 TB/s and, for every round,
//            1.45 (48 rows: 1.85) per 4 tiles of 32 keys and 4.3 (9.6) for every sequence that a range crosses into; those
//            0.84 times with 64 channels
// The constants are a fit to 4,477 calls: 1 to 64 requests, 64 to 40,960 rows of cache, 1 to 64 new tokens, 7 layouts of heads, up
// to 7 ways each. The choice then takes 0.9% longer than the best of them in the mean, 4.8% at the 95th percentile; ranges
// for all calls up to 16 rows, one round of them, and a coarser estimate for more took 19% and 2.3 times. E.g. one token of
// 40 / 8 heads x 128 over 40,688 keys: 32 ranges 41, 0: 452; over 300 keys of 2 requests 5: 12, 0: 9; 64 requests of 512 keys and 3
// tokens 32: 42, 0: 33; of 8,192 keys at most 32: 190, 0: 215.
extern "C" int vdnh3_causal_cached_ranges(int batch, int new_tokens, int room, int heads, int kv_heads, int head_dim) {
  using namespace vdnh3;
  if (batch <= 0 || new_tokens <= 0 || room <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  const int64_t rows = (int64_t)new_tokens * (heads / kv_heads), tiles = batch * (((int64_t)room + kFewKeys - 1) / kFewKeys);
  if (room > kMostRoom || tiles > INT32_MAX || rows * batch > INT32_MAX || rows * batch * kv_heads > INT32_MAX) return 0;
  constexpr double kFull = 0.64;
  const bool narrow = head_dim <= 64;
  const double megabytes = kFull * batch * room * kv_heads * head_dim * 4e-6;
  const double groups = (double)((rows + 127) / 128) * batch * kv_heads;
  double least = 4. + std::max(megabytes / 7.5, (narrow ? 0.75 : 0.9) * std::ceil(groups / 256) * ((room + kBN - 1) / kBN));
  int64_t ranges = 0;
  const int height = few_block(rows);
  const int64_t blocks = (rows + height - 1) / height * kv_heads;
  const double slow = narrow ? 0.84 : 1., step = slow * (height > 32 ? 1.85 : 1.45), cross = slow * (height > 16 ? 9.6 : 4.3);
  for (const int quarters : {0, 1, 2, 4, 8, 12}) {  // of a round; 0: one range
    const int64_t r = std::max<int64_t>(std::min<int64_t>(64 * quarters / blocks, tiles / kFewLeast), 1);
    const double rounds = std::ceil((double)blocks * r / 256), steps = std::ceil(kFull * tiles / (4. * r));
    const double crossings = batch > 1 ? std::max(1., (double)batch / r) : 0.;
    const double us = (height > 16 ? 13. : 10.) - (r == 1 ? 5.3 : 0.) + 0.08 * r / batch + 4.2 * (rounds - 1) +
                      std::max(rounds * (step * steps + cross * crossings), megabytes / 8.);
    if (us < least) least = us, ranges = r;
  }
  return (int)ranges;
}

extern "C" int vdnh3_causal_block_rows(int batch, int new_tokens, int heads, int kv_heads, int head_dim, int ranges) {
  using namespace vdnh3;
  if (batch <= 0 || new_tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || ranges < 0) return 0;
  if (ranges > 0) return few_block((int64_t)new_tokens * (heads / kv_heads));
  return high_blocks(batch, new_tokens, heads, head_dim) ? 256 : 128;
}

extern "C" size_t vdnh3_causal_partial_bytes(int new_tokens, int heads, int head_dim, int ranges) {
  if (new_tokens <= 0 || heads <= 0 || head_dim <= 0 || ranges <= 1) return 0;
  return (size_t)ranges * 2 * new_tokens * heads * (head_dim + 2) * sizeof(float);
}

extern "C" int vdnh3_causal_attn_cached(const uint16_t *q, int64_t q_batch, int64_t q_row, int64_t q_head,
                                        const uint16_t *k, int64_t k_batch, int64_t k_row, int64_t k_head,
                                        const uint16_t *v, int64_t v_batch, int64_t v_row, int64_t v_head, uint16_t *out,
                                        int64_t o_batch, int64_t o_row, int64_t o_head, const int32_t *lengths, int batch,
                                        int new_tokens, int room, int heads, int kv_heads, int head_dim, float scale,
                                        int ranges, float *partial, size_t partial_bytes, void *stream) {
  using namespace vdnh3;
  const Operand qo = operand(q, q_batch, q_row, q_head, batch, new_tokens, heads),
                ko = operand(k, k_batch, k_row, k_head, batch, room, kv_heads),
                vo = operand(v, v_batch, v_row, v_head, batch, room, kv_heads),
                oo = operand(out, o_batch, o_row, o_head, batch, new_tokens, heads);
  int rc = check_causal(qo, ko, vo, oo, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  VDNH3_HOST_CHECK(lengths && batch > 0 && new_tokens > 0 && room > 0, VDNH3_ERR_INVALID,
                   "causal attention: null lengths, or no sequences, new tokens or room in the cache");
  VDNH3_HOST_CHECK(room <= kMostRoom, VDNH3_ERR_INVALID, "causal attention: caches of %d rows are too long", room);
  const Sequences seqs{nullptr, lengths, batch, new_tokens, room};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ranges == 0) return launch_causal(qo, ko, vo, oo, seqs, heads, kv_heads, head_dim, scale, s);
  const int group = heads / kv_heads;
  const int64_t rows = (int64_t)new_tokens * group;
  VDNH3_HOST_CHECK(ranges > 0, VDNH3_ERR_INVALID, "causal attention: the ranges must not be negative, got %d", ranges);
  VDNH3_HOST_CHECK(rows * batch <= INT32_MAX && rows * batch * kv_heads <= INT32_MAX &&
                       (int64_t)batch * (room / kFewKeys + 1) <= INT32_MAX, VDNH3_ERR_INVALID, "causal attention: %d x %d new tokens or caches of %d rows are too many for ranges",
                   batch, new_tokens, room);
  const size_t need = vdnh3_causal_partial_bytes(new_tokens, heads, head_dim, ranges);
  VDNH3_HOST_CHECK(need == 0 || (partial && reinterpret_cast<uintptr_t>(partial) % 16 == 0 && partial_bytes >= need),
                   VDNH3_ERR_INVALID, "causal attention: the ranges' buffer must be 16-byte aligned and hold %zu bytes, got %zu",
                   need, partial_bytes);
  const Parts parts{partial, reinterpret_cast<float2 *>(partial + (size_t)ranges * 2 * new_tokens * heads * head_dim), ranges};
  const float scale_log2 = scale * kLog2E;
  return head_dim == 128 ? launch_few_rows<128>(qo, ko, vo, oo, seqs, kv_heads, group, scale_log2, parts, s)
                         : launch_few_rows<64>(qo, ko, vo, oo, seqs, kv_heads, group, scale_log2, parts, s);
}
