// Causal linear attention with a decay for each head on gfx950, bf16, states fp32: whole prompts of several sequences
// packed one behind another. (New tokens over a pool of states: state_step.hip.)
//
//   S_t = a_h S_{t-1} + v_t k_t^T,   o_t = scale S_t q_t,   a_h = exp(log_decay_h)       S: [dv, dk] per value head h
//
// Value head h reads query / key head h / (heads / qk_heads). Sequence b is the rows [cu[b], cu[b + 1]); its state
// starts from initial[b] or zeros. With chunks of C = 64 tokens that begin with their sequence, row r of a chunk of n:
//   o_r = scale (a^{r+1} S q_r + sum_{j <= r} a^{r-j} (q_r . k_j) v_j),   S' = a^n S + sum_j a^{n-1-j} v_j k_j^T
//
// All three are bf16 MFMA with fp32 sums. Against rounding, S and the scores meet their products as two bf16 numbers (2^-17; one
// would add 2^-9 of them to the outputs' own 2^-9), the weighted values as three: the states keep 24 bits.
// Chunks of a sequence follow one another, so a head's chunks are cut into ranges that run beside each other, a workgroup a CU: a
// first pass makes the state that each range adds, and the second starts from them. It reads K and V twice.
// 40,688 tokens x 40 heads x 128 take 610 to 625 us: the first pass 185 (its loads alone 141, its arithmetic alone 150), the second
// 425 (loads and stores alone 330, arithmetic alone 345): 106 chunks of 4.0 us, by the counters 7,830 cycles at 2.0 GHz, of which a
// SIMD's matrix core is busy 3,105 and its vector unit 4,096, each wavefront now in one, now in the other. 3,939 tokens of 7
// sequences take 80 us, 512 of one 29, 77 13.7 (a launch, a start of three loads one after another, two chunks).
#include <algorithm>
#include <cmath>

#include "common.h"

namespace vdnh3 {
namespace {

constexpr int kLinC = 64;  // tokens of a chunk

struct LinOperand {
  const uint16_t *p;
  int64_t row, head;
};

struct LinCall {
  LinOperand q, k, v;
  uint16_t *out;
  int64_t o_row, o_head;
  const float *log_decay;
  const int32_t *cu;
  const float *initial;
  float *final_state;
  float *carry;    // [ranges, heads, D, D]: the state at the end of a range, where its last sequence goes on
  int32_t *meta;   // [ranges]: tokens of a range that lies in one sequence begun before it, -1 for others
  int sequences, rows, heads, group, ranges;
  int scanned;     // the states at the ranges' ends are whole, not only what each range adds
  float scale;
};

// a^n of a head from log2 a. 0 * -inf (a head that keeps nothing) is 1 here.
__device__ __forceinline__ float decay_pow(float log2a, int n) {
  return n == 0 ? 1.f : __builtin_amdgcn_exp2f(log2a * (float)n);
}

__device__ __forceinline__ int lin_bound(const LinCall &p, int b) { return min(max(p.cu[b], 0), p.rows); }

// Where a workgroup is: sequence b (rows [s0, s1)), the chunk that begins at row `row` of q, k and v.
struct LinPlace {
  int b, s0, s1, row;
};

// The workgroup's range of the chunks of all sequences, one sequence behind another: equal ranges, whatever the lengths, and
// none empty in front of one that is not. Every thread adds up the chunks of sequences next to each other; the one that has the
// range's first chunk finds its sequence. `count` chunks begin at `at`.
struct LinRange {
  int64_t count;
  LinPlace at;
};
template <int THREADS>
__device__ __forceinline__ LinRange lin_range(const LinCall &p, int range, int64_t *sums, int *found) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (p.sequences + THREADS - 1) / THREADS;
  const int b0 = (int)min((int64_t)tid * per, (int64_t)p.sequences), b1 = min(b0 + per, p.sequences);
  auto chunks_of = [&](int b, int &s, int &e) __device__ {
    s = lin_bound(p, b);
    e = max(lin_bound(p, b + 1), s);
    return (e - s + kLinC - 1) / kLinC;
  };
  int64_t mine = 0;
  int s, e;
  for (int b = b0; b < b1; ++b) mine += chunks_of(b, s, e);
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t x = __shfl_up(upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) upto += sums[w];
    total += sums[w];
  }
  const int64_t ranges = min((int64_t)p.ranges, total);
  if (range >= ranges) return LinRange{0, LinPlace{0, 0, 0, 0}};
  const int64_t c0 = total * range / ranges, c1 = total * (range + 1) / ranges;
  int64_t c = c0 - (upto - mine);
  if (c >= 0 && c0 < upto) {
    int b = b0, n = chunks_of(b, s, e);
    while (c >= n) {  // the thread's sequences hold more than c chunks
      c -= n;
      n = chunks_of(++b, s, e);
    }
    found[0] = b;
    found[1] = s;
    found[2] = e;
    found[3] = s + (int)c * kLinC;
  }
  __syncthreads();
  return LinRange{c1 - c0, LinPlace{__builtin_amdgcn_readfirstlane(found[0]), __builtin_amdgcn_readfirstlane(found[1]),
                                    __builtin_amdgcn_readfirstlane(found[2]), __builtin_amdgcn_readfirstlane(found[3])}};
}

// LDS slots: chunk c (16 bytes) of row r lies at slot c ^ swizzle(r). Four neighbouring chunks of four neighbouring rows
// (transposed reads) lie in 16 different 16-byte bank groups; so do the chunks 4 t + g of the rows that one turn of a 16-byte
// fragment read takes, rows 0 to 3 and 12 to 15 of one g with rows 4 to 11 of the next (8 cycles a wavefront with r / 4 for 0, 2,
// 3, 1: 6).
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  const int four = ((r ^ (r >> 1)) & 4) >> 1 | ((r >> 3) & 1);  // 0, 2, 3, 1 for r / 4 = 0, 1, 2, 3
  if constexpr (D == 128) return ((r & 3) << 2) | four;
  else return (((r >> 1) & 1) << 2) | four;
}

typedef short lin_s16x4_t __attribute__((ext_vector_type(4)));
// Four rows of one channel per lane: 16 lanes read 4 rows of 16 channels (lane i: 4 channels of row i / 4) and get their
// transpose (lane i: channel i of the 4 rows).
__device__ __forceinline__ u32x2_t lin_read_transposed(const uint16_t *p) {
  typedef __attribute__((address_space(3))) lin_s16x4_t *lds_ptr;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p)));
}

__device__ __forceinline__ float lo_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// What the halves of a pair of bf16 numbers leave of the number that they were rounded from, exactly
__device__ __forceinline__ float rest_lo(uint32_t hi, float x) { return x - lo_half(hi); }
__device__ __forceinline__ float rest_hi(uint32_t hi, float x) { return x - hi_half(hi); }
// x as two bf16 numbers each that hold 16 bits of it
struct Split2 {
  u32x4_t hi, lo;
};
__device__ __forceinline__ Split2 split2(const float *x) {
  Split2 s;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s.hi[j] = pack_bf2(x[2 * j], x[2 * j + 1]);
    s.lo[j] = pack_bf2(rest_lo(s.hi[j], x[2 * j]), rest_hi(s.hi[j], x[2 * j + 1]));
  }
  return s;
}
// Whether one of eight bf16 numbers is an infinity or a NaN: only their |x| of 0x7f80 and more reach bit 15 with 0x80 more
__device__ __forceinline__ bool has_wild(u32x4_t x) {
  x = (x & 0x7fff7fffu) + 0x00800080u;
  return ((x[0] | x[1] | x[2] | x[3]) & 0x80008000u) != 0;
}

// A workgroup of D / 16 wavefronts walks a range of a head's chunks; a wavefront carries 16 rows (dv) of the state in
// accumulators, as C[dk][dv] tiles: row 4 g + i of tile t is dk = 32 (t / 2) + 8 g + 4 (t % 2) + i, so that two tiles are the
// operand of S q as they lie, a lane with eight neighbouring dk of its dv. Outputs are computed transposed, O^T[dv][row].
// CARRY: only the state at the range's end, where the last sequence goes on behind it.
template <int D, bool CARRY>
__global__ __launch_bounds__(D * 4, 1) void causal_linear_kernel(LinCall p) {
  constexpr int C = kLinC, KC = D / 8, NW = D / 16, THREADS = 64 * NW, TILE = C * D;
  constexpr int NS = D / 32;            // k-steps over dk
  constexpr int PT = NW == 8 ? 2 : 4;   // 16 x 16 tiles of P that a wavefront makes at most
  // Tiles on their way two chunks ahead where LDS holds three of each (156 KB; one ahead 625 us for 610), else one (two
  // workgroups a CU). The first pass gains nothing by a third.
  constexpr int RING = D == 128 && !CARRY ? 3 : 2, LOADS = (CARRY ? 2 : 3) * C * KC / THREADS;
  __shared__ __attribute__((aligned(16))) uint16_t Ks[RING][TILE], Vs[RING][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t Qs[CARRY ? 1 : RING][CARRY ? 8 : TILE];
  __shared__ __attribute__((aligned(16))) u32x4_t Ps[CARRY ? 1 : 2][CARRY ? 1 : 6][64];  // hi / lo, (row tile, k-step), lane
  __shared__ int64_t sums[NW];
  __shared__ int found[4];

  const int h = (int)blockIdx.x % p.heads, range = (int)blockIdx.x / p.heads, hk = h / p.group;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const float log2a = p.log_decay[h] * 1.44269504088896341f;
  LinRange rg = lin_range<THREADS>(p, range, sums, found);
  const int dv = 16 * wave + l16;  // the lane's row of the state

  // ---- states between memory and the accumulators -----------------------------------------------------------------
  f32x4_t s[D / 16];
  auto load_state = [&](const float *from) __device__ {
    if (from == nullptr) {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) s[t] = f32x4_t{};
      return;
    }
    const float *r = from + (int64_t)dv * D + 8 * g;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) s[t] = *reinterpret_cast<const f32x4_t *>(r + 16 * t - 12 * (t % 2));
    // here, once a sequence: left to the loop, the wait for them is one for every load and store of each chunk
#pragma unroll
    for (int t = 0; t < D / 16; ++t) asm volatile("" : "+v"(s[t]));
  };
  auto store_state = [&](float *to) __device__ {
    float *r = to + (int64_t)dv * D + 8 * g;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4_t *>(r + 16 * t - 12 * (t % 2)) = s[t];
  };
  const int64_t state_at = (int64_t)h * D * D, state_step = (int64_t)p.heads * D * D;
  auto initial_of = [&](int b) __device__ { return p.initial ? p.initial + b * state_step + state_at : nullptr; };
  // empty sequences from b on end as they began; the first that is not empty
  auto pass_empty = [&](int b) __device__ {
    for (; b < p.sequences && lin_bound(p, b + 1) <= lin_bound(p, b); ++b) {
      if (CARRY || !p.final_state) continue;
      const float *from = initial_of(b);
      float *to = p.final_state + b * state_step + state_at;
      for (int i = 4 * tid; i < D * D; i += 4 * THREADS)
        *reinterpret_cast<f32x4_t *>(to + i) = from ? *reinterpret_cast<const f32x4_t *>(from + i) : f32x4_t{};
    }
    return b;
  };

  if (CARRY) {
    if (tid == 0 && h == 0) p.meta[range] = -1;
    if (rg.count <= 0) return;
    // the range's last chunk and the sequence that it is of; nothing to do where that ends here
    LinPlace at = rg.at;
    int64_t left = rg.count;
    bool open = at.row > at.s0;
    while (true) {
      const int chunks = (at.s1 - at.row + C - 1) / C;
      if (chunks == left) return;
      if (chunks > left) break;
      left -= chunks;
      int b = at.b + 1;
      while (lin_bound(p, b + 1) <= lin_bound(p, b)) ++b;  // there is a chunk left, so one of them is not empty
      at = LinPlace{b, lin_bound(p, b), lin_bound(p, b + 1), lin_bound(p, b)};
      open = false;
    }
    rg = LinRange{left, at};
    if (tid == 0 && h == 0 && open) p.meta[range] = (int)left * C;
    load_state(open ? nullptr : initial_of(at.b));
  } else {
    if (range == 0) pass_empty(0);
    if (rg.count <= 0) return;
    if (rg.at.row == rg.at.s0) {
      load_state(initial_of(rg.at.b));
    } else {
      int w = range - 1;
      load_state(p.carry + w * state_step + state_at);
      // where nobody has: what the ranges in front add to it, back to the one in which the sequence begins
      float fade = 1.f;
      for (int tokens; w > 0 && !p.scanned && (tokens = p.meta[w]) >= 0;) {
        fade *= decay_pow(log2a, tokens);
        const float *r = p.carry + --w * state_step + state_at + (int64_t)dv * D + 8 * g;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t *>(r + 16 * t - 12 * (t % 2));
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][i] = fmaf(fade, x[i], s[t][i]);
        }
      }
    }
  }

  // ---- tile loads, straight to LDS: thread chunk i fills position THREADS i + tid: row P / KC, slot P % KC ----------
  constexpr int CG = C * KC / THREADS;
  static_assert(CG == 2 && THREADS / KC % 16 == 0, "the swizzle is the same for a thread's rows");
  const int kr0 = tid / KC, slot16 = tid % KC;
  const uint32_t chunk = (slot16 ^ swizzle<D>(kr0)) * 8;
  const uint16_t *kp = p.k.p + hk * p.k.head, *vp = p.v.p + h * p.v.head, *qp = p.q.p + hk * p.q.head;
  const uint32_t wave_lds = __builtin_amdgcn_readfirstlane(wave * 1024);
  // rows behind the chunk's last repeat it: their weights are zero and their outputs are not stored
  uint32_t k_off[CG], v_off[CG], q_off[CG];
#pragma unroll
  for (int i = 0; i < CG; ++i) {
    const uint32_t r = kr0 + i * (THREADS / KC);
    k_off[i] = 2u * (r * (uint32_t)p.k.row + chunk);
    v_off[i] = 2u * (r * (uint32_t)p.v.row + chunk);
    q_off[i] = 2u * (r * (uint32_t)p.q.row + chunk);
  }
  auto load_tile = [&](const uint16_t *base, int64_t stride, const uint32_t *whole, int n, const uint16_t *tile) __device__ {
    uint32_t off[CG];
#pragma unroll
    for (int i = 0; i < CG; ++i)
      off[i] = n == C ? whole[i] : 2u * ((uint32_t)min(kr0 + i * (THREADS / KC), n - 1) * (uint32_t)stride + chunk);
#pragma unroll
    for (int i = 0; i < CG; ++i) global_to_lds16_sbase(base, off[i], lds_address(tile) + wave_lds + i * THREADS * 16);
  };
  auto load_tiles = [&](const LinPlace &place, int slot) __device__ {
    const int n = min(C, place.s1 - place.row);
    const int64_t row = place.row;
    load_tile(kp + row * p.k.row, p.k.row, k_off, n, Ks[slot]);
    load_tile(vp + row * p.v.row, p.v.row, v_off, n, Vs[slot]);
    if constexpr (!CARRY) load_tile(qp + row * p.q.row, p.q.row, q_off, n, Qs[slot]);
  };

  // ---- what stays the same over a head's chunks ----------------------------------------------------------------------
  // fragments of row l16 of a 16-row tile of Q or K by 32 dk; transposed reads of K by a pair of dk tiles, and of V
  int qk_at[NS], kt_at[NS];
  const int tr = 4 * g + (l16 >> 2);
  auto tile_at = [&](int r, int c) __device__ { return r * D + (c ^ swizzle<D>(r)) * 8; };
#pragma unroll
  for (int t = 0; t < NS; ++t) {
    qk_at[t] = tile_at(l16, 4 * t + g);
    kt_at[t] = tile_at(tr, 4 * t + (l16 & 3));
  }
  auto qk_frag = [&](const uint16_t *tile, int t) __device__ { return as_bf16x8(ld16(tile + qk_at[t])); };
  const int vt_at = tile_at(tr, 2 * wave + ((l16 >> 1) & 1)) + 4 * (l16 & 1);
  // the wavefront's tiles of P^T: row tile prt, token tiles pu, pu + PS, ... up to the diagonal
  constexpr int PS = NW / 4;
  const int prt = wave / PS, pu = wave % PS;
  float pw[PT][4], row_weight[4];
  if constexpr (!CARRY) {
#pragma unroll
    for (int x = 0; x < PT; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) pw[x][i] = p.scale * decay_pow(log2a, max(16 * (prt - pu - PS * x) + l16 - 4 * g - i, 0));
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) row_weight[rt] = p.scale * decay_pow(log2a, 16 * rt + l16 + 1);
    // tiles of P behind the diagonal that share a k-step with one on it
    for (int i = tid; i < 2 * 6 * 64; i += THREADS) (&Ps[0][0][0])[i] = u32x4_t{};
  }
  float vw[16];  // a^{n-1-j} of the lane's tokens j of a chunk of n
  int vw_n = -1;

  // the next chunk of the range
  auto after = [&](const LinPlace &place) __device__ {
    if (place.row + C < place.s1) return LinPlace{place.b, place.s0, place.s1, place.row + C};
    const int b = pass_empty(place.b + 1);
    return LinPlace{b, lin_bound(p, b), lin_bound(p, b + 1), lin_bound(p, b)};
  };
  // P^T = scale K Q^T with the decays, as two bf16 numbers
  auto make_p = [&](const uint16_t *kt, const uint16_t *qt) __device__ {
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      const int u = pu + PS * x;
      if (u > prt) break;
      f32x4_t c = {};
#pragma unroll
      for (int t = 0; t < NS; ++t) c = mfma_bf16_16x16x32(qk_frag(kt + 16 * u * D, t), qk_frag(qt + 16 * prt * D, t), c);
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // behind the diagonal nothing is taken, whatever the key holds
        w[i] = u < prt || l16 >= 4 * g + i ? c[i] * pw[x][i] : 0.f;
      }
      const uint32_t h0 = pack_bf2(w[0], w[1]), h1 = pack_bf2(w[2], w[3]);
      const uint32_t e0 = pack_bf2(rest_lo(h0, w[0]), rest_hi(h0, w[1])), e1 = pack_bf2(rest_lo(h1, w[2]), rest_hi(h1, w[3]));
      const int f = prt < 2 ? prt : 2 * prt - 2 + (u >> 1);
      reinterpret_cast<u32x2_t *>(&Ps[0][f][lane])[u & 1] = u32x2_t{h0, h1};
      reinterpret_cast<u32x2_t *>(&Ps[1][f][lane])[u & 1] = u32x2_t{e0, e1};
    }
  };

  // the wavefronts of a SIMD (w and w + 4) at different steps, one at the matrix core and one at the vector unit (606 us, 610)
  if (!CARRY && NW == 8 && wave >= 4) __builtin_amdgcn_s_setprio(1);
  LinPlace at = rg.at, next = at;
  int slot = 0, o_row = 0, o_n = 0;
  // outputs lie in the Q tile of their chunk, which no wavefront reads any more, until they are stored in whole rows
  auto store_outputs = [&](const uint16_t *tile) __device__ {
#pragma unroll
    for (int i = 0; i < CG; ++i) {
      const int r = kr0 + i * (THREADS / KC);
      if (r < o_n) st16(p.out + (int64_t)(o_row + r) * p.o_row + h * p.o_head + chunk, ld16(tile + (r * KC + slot16) * 8));
    }
  };
  load_tiles(at, 0);
  if (rg.count > 1) {
    next = after(at);
    if (RING == 3) load_tiles(next, 1);
  }
  for (int64_t left = rg.count; left > 0; --left) {
    const int slot_next = slot + 1 == RING ? 0 : slot + 1, slot_last = slot == 0 ? RING - 1 : slot - 1;
    // this chunk's tiles; the next one's, the newest that were asked for, may still be on their way
    if (RING == 3 && left > 1) wait_vm_lds<LOADS>();
    else wait_vm_lds<0>();
    bare_barrier();
    const int n = min(C, at.s1 - at.row);
    const bool ends = at.row + C >= at.s1;
    LinPlace later = next;  // the chunk after the next
    if (left > 2) later = after(next);
    if (RING == 2 && left > 1) load_tiles(next, slot_next);
    if (RING == 3 && !CARRY) store_outputs(Qs[CARRY ? 0 : slot_last]);
    if (!CARRY && ends && left == 1) pass_empty(at.b + 1);

    if (n != vw_n) {
      vw_n = n;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int back = n - 1 - (16 * (x / 4) + 4 * g + x % 4);
        vw[x] = back < 0 ? 0.f : decay_pow(log2a, back);
      }
    }
    const uint16_t *kt = Ks[slot], *vt = Vs[slot];
    u32x4_t vf[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const u32x2_t a = lin_read_transposed(vt + 32 * ks * D + vt_at), b = lin_read_transposed(vt + (32 * ks + 16) * D + vt_at);
      vf[ks] = u32x4_t{a[0], a[1], b[0], b[1]};
    }

    if constexpr (!CARRY) {
      uint16_t *qt = Qs[slot];
      make_p(kt, qt);
      // O^T = S Q^T, rows by scale a^{r+1}
      f32x4_t o[4] = {};
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[2 * t + j / 4][j % 4];
        const Split2 sp = split2(x);
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          const bf16x8_t qf = qk_frag(qt + 16 * rt * D, t);
          o[rt] = mfma_bf16_16x16x32(as_bf16x8(sp.hi), qf, o[rt]);
          o[rt] = mfma_bf16_16x16x32(as_bf16x8(sp.lo), qf, o[rt]);
        }
      }
#pragma unroll
      for (int rt = 0; rt < 4; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[rt][i] *= row_weight[rt];
      // a value that is no finite number would reach rows in front of it as 0 * inf: it is left out of the product, and its
      // channel ends there
      const bool careful = __any(has_wild(vf[0]) || has_wild(vf[1]));
      u32x4_t vc[2] = {vf[0], vf[1]};
      int bad = C;
      if (careful) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t mask = j & 1 ? 0xffff0000u : 0xffffu, most = j & 1 ? 0x7f800000u : 0x7f80u;
            if ((vf[ks][j / 2] & most) == most) {
              bad = min(bad, 32 * ks + 16 * (j / 4) + 4 * g + j % 4);
              vc[ks][j / 2] &= ~mask;
            }
          }
        bad = min(bad, __shfl_xor(bad, 16));
        bad = min(bad, __shfl_xor(bad, 32));
      }
      wait_vm_lds<63>();
      bare_barrier();
#pragma unroll
      for (int rt = 0; rt < 4; ++rt)
#pragma unroll
        for (int ks = 0; ks <= rt / 2; ++ks) {
          const int f = rt < 2 ? rt : 2 * rt - 2 + ks;
          o[rt] = mfma_bf16_16x16x32(as_bf16x8(vc[ks]), as_bf16x8(Ps[0][f][lane]), o[rt]);
          o[rt] = mfma_bf16_16x16x32(as_bf16x8(vc[ks]), as_bf16x8(Ps[1][f][lane]), o[rt]);
        }
      if (careful) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = __shfl(bad, 4 * g + i);
#pragma unroll
          for (int rt = 0; rt < 4; ++rt)
            if (16 * rt + l16 >= from) o[rt][i] = __builtin_nanf("");
        }
      }
      if constexpr (RING == 3) {
        // chunk c of row r at slot c ^ swizzle(r), as Q's
#pragma unroll
        for (int rt = 0; rt < 4; ++rt)
          *reinterpret_cast<u32x2_t *>(qt + 16 * rt * D + tile_at(l16, 2 * wave + (g >> 1)) + 4 * (g & 1)) =
              u32x2_t{pack_bf2(o[rt][0], o[rt][1]), pack_bf2(o[rt][2], o[rt][3])};
        o_row = at.row;
        o_n = n;
        if (left > 2) load_tiles(later, slot_last);
      } else {
        uint16_t *op = p.out + (int64_t)at.row * p.o_row + h * p.o_head + 16 * wave + 4 * g;
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          const int r = 16 * rt + l16;
          if (r < n)
            *reinterpret_cast<u32x2_t *>(op + r * p.o_row) = u32x2_t{pack_bf2(o[rt][0], o[rt][1]), pack_bf2(o[rt][2], o[rt][3])};
        }
      }
    }

    // S' = a^n S + K^T V, the weighted values as three bf16 numbers, which hold them whole
    const float all = decay_pow(log2a, n);
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] *= all;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4_t w[3];
      bf16x8_t kf[D / 16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x0 = lo_half(vf[ks][j]) * vw[8 * ks + 2 * j], x1 = hi_half(vf[ks][j]) * vw[8 * ks + 2 * j + 1];
        w[0][j] = pack_bf2(x0, x1);
        const float y0 = rest_lo(w[0][j], x0), y1 = rest_hi(w[0][j], x1);
        w[1][j] = pack_bf2(y0, y1);
        w[2][j] = pack_bf2(rest_lo(w[1][j], y0), rest_hi(w[1][j], y1));
      }
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const uint16_t *kr = kt + 32 * ks * D + kt_at[t / 2] + 4 * (t % 2);
        const u32x2_t a = lin_read_transposed(kr), b = lin_read_transposed(kr + 16 * D);
        kf[t] = as_bf16x8(u32x4_t{a[0], a[1], b[0], b[1]});
      }
      // four tiles in turn: a product waits for the last one into the same tile
#pragma unroll
      for (int t = 0; t < D / 16; t += 4)
#pragma unroll
        for (int e = 2; e >= 0; --e)
#pragma unroll
          for (int u = t; u < t + 4; ++u) s[u] = mfma_bf16_16x16x32(kf[u], as_bf16x8(w[e]), s[u]);
    }
    if (!CARRY && ends) {
      if (p.final_state) store_state(p.final_state + at.b * state_step + state_at);
      if (left > 1) load_state(initial_of(next.b));
    }
    at = next;
    next = later;
    slot = slot_next;
  }
  if constexpr (RING == 3 && !CARRY) {
    wait_vm_lds<63>();
    bare_barrier();
    store_outputs(Qs[slot == 0 ? RING - 1 : slot - 1]);
  }
  if (CARRY) store_state(p.carry + range * state_step + state_at);
}

// The states at the ranges' ends from those that each range adds: carry[w] += a^{tokens of w} carry[w - 1] where range w lies
// in a sequence that began before it. Four numbers a thread, range after range.
__global__ __launch_bounds__(256) void carry_scan_kernel(LinCall p, int numbers) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, all = (int64_t)p.heads * numbers;
  if (i >= all) return;
  const float log2a = p.log_decay[i / numbers] * 1.44269504088896341f;
  f32x4_t acc = *reinterpret_cast<const f32x4_t *>(p.carry + i);
  for (int w = 1; w + 1 < p.ranges; ++w) {
    float *at = p.carry + w * all + i;
    f32x4_t x = *reinterpret_cast<const f32x4_t *>(at);
    const int tokens = p.meta[w];
    if (tokens >= 0) {
      const float a = decay_pow(log2a, tokens);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = fmaf(a, acc[j], x[j]);
      *reinterpret_cast<f32x4_t *>(at) = x;
    }
    acc = x;
  }
}

template <int D>
int launch_causal_linear(const LinCall &p, hipStream_t s) {
  if (p.ranges > 1) {
    hipLaunchKernelGGL((causal_linear_kernel<D, true>), dim3(p.ranges * p.heads), dim3(D * 4), 0, s, p);
    int rc = check_launch("causal_linear");
    if (rc) return rc;
    if (p.scanned) {
      const int64_t groups = ((int64_t)p.heads * D * D / 4 + 255) / 256;
      hipLaunchKernelGGL(carry_scan_kernel, dim3((unsigned)groups), dim3(256), 0, s, p, D * D);
      rc = check_launch("causal_linear");
      if (rc) return rc;
    }
  }
  hipLaunchKernelGGL((causal_linear_kernel<D, false>), dim3(p.ranges * p.heads), dim3(D * 4), 0, s, p);
  return check_launch("causal_linear");
}

// Up to so many ranges each adds up what those in front of it left, its workgroups for themselves; more take a launch of their
// own for it (9 ranges of 56 heads x 64: 83 us and 86, 4 of 40 x 128 28.8 and 30.1, 6 of 7 sequences 80 and 84; 32 of 8 heads 87
// and 57).
constexpr int kAddedRanges = 16;

// Chunks of a call, at most: the sequences' lengths are on the device.
int64_t most_chunks(int64_t rows, int64_t sequences) { return rows / kLinC + std::min(rows, sequences); }

int check_lin_operand(const void *p, int64_t row, int64_t head, const char *name) {
  VDNH3_HOST_CHECK(p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && head % 8 == 0 && row >= 0 &&
                       head >= 0 && row <= (1 << 23),
                   VDNH3_ERR_INVALID, "causal_linear: %s must be 16-byte aligned with strides that are multiples of 8, rows at "
                   "most 2^23 elements apart", name);
  return VDNH3_OK;
}

}  // namespace
}  // namespace vdnh3

extern "C" int vdnh3_causal_linear_ranges(int rows, int sequences, int heads, int head_dim) {
  if (rows <= 0 || sequences <= 0 || heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  // One round of workgroups, two chunks of each or more: 512 tokens x 40 heads x 128 take 29 us in 4 ranges (1 33, 3 31, 6 33),
  // 3,939 of 7 sequences 80 in 6 (5 90, 12 91, 1 247), 40,688 610 (4 780, 12 620, 1 2,070); 8,000 x 56 x 64 87 in 9 (4 124, 18
  // 101).
  const int64_t slots = head_dim == 128 ? 256 : 512;  // workgroups that run at once
  return (int)std::max<int64_t>(1, std::min(slots / heads, vdnh3::most_chunks(rows, sequences) / 2));
}

extern "C" size_t vdnh3_causal_linear_workspace_bytes(int ranges, int heads, int head_dim) {
  if (ranges <= 1 || heads <= 0 || head_dim <= 0) return 0;
  return (size_t)ranges * heads * head_dim * head_dim * 4 + (size_t)ranges * 4;
}

extern "C" int vdnh3_causal_linear_packed(const uint16_t *q, int64_t q_row, int64_t q_head, const uint16_t *k, int64_t k_row,
                                          int64_t k_head, const uint16_t *v, int64_t v_row, int64_t v_head, uint16_t *out,
                                          int64_t o_row, int64_t o_head, const float *log_decay, const int32_t *cu_seqlens,
                                          const float *initial_state, float *final_state, int sequences, int rows,
                                          int heads, int qk_heads, int head_dim, float scale, int ranges, void *workspace,
                                          size_t workspace_bytes, void *stream) {
  using namespace vdnh3;
  VDNH3_HOST_CHECK(head_dim == 64 || head_dim == 128, VDNH3_ERR_INVALID, "causal_linear: head_dim must be 64 or 128, got %d",
                   head_dim);
  VDNH3_HOST_CHECK(rows > 0 && sequences > 0 && heads > 0 && qk_heads > 0 && heads % qk_heads == 0, VDNH3_ERR_INVALID,
                   "causal_linear: rows, sequences and heads must be positive and heads a multiple of qk_heads, got %d rows, "
                   "%d sequences, %d / %d heads", rows, sequences, heads, qk_heads);
  // one row, or one head, has no stride, whatever a caller passes for it
  if (rows == 1) q_row = k_row = v_row = o_row = 0;
  if (qk_heads == 1) q_head = k_head = 0;
  if (heads == 1) v_head = o_head = 0;
  int rc = check_lin_operand(q, q_row, q_head, "q");
  if (!rc) rc = check_lin_operand(k, k_row, k_head, "k");
  if (!rc) rc = check_lin_operand(v, v_row, v_head, "v");
  if (!rc) rc = check_lin_operand(out, o_row, o_head, "out");
  if (rc) return rc;
  VDNH3_HOST_CHECK(log_decay && cu_seqlens, VDNH3_ERR_INVALID, "causal_linear: decays and sequence bounds are needed");
  VDNH3_HOST_CHECK(reinterpret_cast<uintptr_t>(initial_state) % 16 == 0 && reinterpret_cast<uintptr_t>(final_state) % 16 == 0,
                   VDNH3_ERR_INVALID, "causal_linear: states must be 16-byte aligned");
  VDNH3_HOST_CHECK(std::isfinite(scale), VDNH3_ERR_INVALID, "causal_linear: scale must be finite");
  VDNH3_HOST_CHECK(ranges >= 1 && ranges <= (1 << 20), VDNH3_ERR_INVALID, "causal_linear: ranges must be positive, got %d",
                   ranges);
  VDNH3_HOST_CHECK(ranges == 1 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                                   workspace_bytes >= vdnh3_causal_linear_workspace_bytes(ranges, heads, head_dim)),
                   VDNH3_ERR_INVALID, "causal_linear: %d ranges need a 16-byte aligned workspace of %zu bytes", ranges,
                   vdnh3_causal_linear_workspace_bytes(ranges, heads, head_dim));
  VDNH3_HOST_CHECK((int64_t)rows + sequences < (1ll << 31) - 64, VDNH3_ERR_INVALID, "causal_linear: %d rows are too many", rows);
  rc = check_grid((int64_t)ranges * heads, head_dim * 4, "causal_linear");
  if (!rc) rc = check_grid((int64_t)heads * head_dim * head_dim / 1024, 256, "causal_linear");
  if (rc) return rc;
  float *carry = static_cast<float *>(workspace);
  const LinCall p{{q, q_row, q_head}, {k, k_row, k_head}, {v, v_row, v_head}, out, o_row, o_head, log_decay, cu_seqlens,
                  initial_state, final_state, carry,
                  reinterpret_cast<int32_t *>(carry + (ranges > 1 ? (int64_t)ranges * heads * head_dim * head_dim : 0)),
                  sequences, rows, heads, heads / qk_heads, ranges, ranges > kAddedRanges, scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return head_dim == 128 ? launch_causal_linear<128>(p, s) : launch_causal_linear<64>(p, s);
}
