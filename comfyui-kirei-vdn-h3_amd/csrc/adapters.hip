// Low-rank adapters of many requests beside a shared projection on gfx950, bf16:
//
//   out_t = bf16(y_t + s_i B_i (A_i x_t)),  i = index[t]     A_i: [rank, width], B_i: [out_width, rank], s_i fp32
//
// y is the projection's output for all rows; a row whose index names no adapter keeps it. h = A x is held in fp32, summed over
// the parts of the width that a workgroup's wavefronts take; s h meets B as two bf16 numbers (16 bits of it), and the sum with y
// is rounded once. Rows are taken in blocks of 16 to 64 neighbours; a block finds the adapters in it by ballots and takes their
// rows together, so the rows of one request share each fragment of its adapter, in whatever order requests lie.
//
// A and B are kept in the order in which the wavefronts read them, a kilobyte of neighbours per load: fragments of 16 ranks x 32
// channels of A (strided rows of A took 18 us of 31 at 3,939 rows x 5,120 of rank 32) and of 32 columns x 32 (16) ranks of B.
// x, y and out move in runs of 128 bytes of a row. 40,688 rows x 5,120 -> 5,120 of rank 64, each row with an adapter, take 304 us:
// the first product alone 105 (x, 4.0 TB/s; behind the second, whose last outputs are still on their way to HBM, 127), the second
// alone 192 (y and out, 4.3 TB/s, where a large copy reaches 4.8). Rows that name no adapter are copied: 257 us with a third of
// them, 209 with two. Adapters that change from row to row take 531. One row x 5,120 -> 15,360 of rank 16: 6.0 us in one launch, a
// chain of loads.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace vdnh3 {
namespace {

constexpr int kListRows = 64;    // the most rows of a block
constexpr int kExpandRows = 32;  // 64 leave one wavefront a SIMD: 40,688 rows x 5,120 of rank 64 take 700 us instead of 304
constexpr int kShrinkWaves = 8;
constexpr int kFewRows = 64, kFewRanks = 64;  // up to which one launch can make both products

struct AdapterCall {
  const uint16_t *x, *y, *down, *up;
  uint16_t *out;
  int64_t x_row, y_row, out_row;
  const float *scales;
  const int32_t *index;
  uint16_t *h;  // [rows, ranks, in eights: 8 first numbers, 8 second ones]: s A x as two bf16 numbers
  int rows, width, out_width, adapters, rank, ranks, shares, copy;  // ranks: 16, or the rank rounded up to 32
};

// Between what lanes of a wavefront write to LDS and what others of them read: its LDS operations run in order, but the compiler
// may leave out or move accesses of which no lane's own reads tell.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The adapter of each of a block's rows, a lane a row: -1 for none and behind the last row.
__device__ __forceinline__ int adapter_of(const AdapterCall &p, int row0, int block_rows) {
  const int lane = threadIdx.x & 63;
  const int i = lane < block_rows && row0 + lane < p.rows ? p.index[row0 + lane] : -1;
  return i >= 0 && i < p.adapters ? i : -1;
}

// The rows of `mask`, one behind another, as a wavefront's list; the last one repeats behind its end.
__device__ __forceinline__ void list_rows(uint64_t mask, int *list) {
  const int lane = threadIdx.x & 63, at = __popcll(mask & ((1ull << lane) - 1)), count = __popcll(mask);
  wave_sync();
  if ((mask >> lane) & 1) list[at] = lane;
  if (lane >= count) list[lane] = 63 - __builtin_clzll(mask);
  wave_sync();
}

// What the first bf16 number of x, `hi` as fp32 bits, leaves of it: nothing of an infinity, where inf - inf is a NaN
__device__ __forceinline__ float rest(float x, uint32_t hi) {
  const float d = x - __uint_as_float(hi);
  return d == d ? d : 0.f;
}

// s A x of the rows of one adapter in a block, in two bf16 numbers, 2^-17 of it: one would add 1.1e-3 of the product to the
// result's own 1.7e-3 of rounding. The wavefronts take steps of 64 channels in turn and add their sums up in LDS.
// C[rank][row] tiles: a lane has four ranks of a row.
// `h` holds the rows of the list one behind another (LISTED), or all rows.
template <int MT, int NT, bool LISTED>
__device__ __forceinline__ void shrink_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int rank0,
                                            u32x4_t (*sums)[64], uint16_t *h) {
  constexpr int T = MT * NT, W = kShrinkWaves, TURN = T < W ? T : W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int steps = (p.width + 63) / 64, tiles16 = p.ranks / 16, r8 = lane >> 3, c8 = lane & 7;
  // x is read in runs of 128 bytes of a row, eight rows at a time, and turns into fragments in the wavefront's part of LDS:
  // chunk c (16 bytes) of row r lies at slot c ^ (r % 8)
  u32x4_t *stage = &sums[0][0] + wave * (16 * MT * 8);
  const uint16_t *xp[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) xp[i] = p.x + (int64_t)(row0 + list[8 * i + r8]) * p.x_row;
  // ranks behind the last tile read it again; their sums are not used
  const uint16_t *ap = p.down + ((int64_t)adapter * steps * tiles16 + rank0 / 16) * 1024 + lane * 8;
  const int most = tiles16 - rank0 / 16 - 1;
  f32x4_t acc[T] = {};
  __syncthreads();  // the sums of another adapter have been read
  for (int step = wave; step < steps; step += W) {
    u32x4_t a[2][NT], x[2 * MT];
    // channels behind the width: A holds zeros for them, and x, read again, becomes zeros (0 * inf would be a NaN)
    const int c = 64 * step + 8 * c8;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) x[i] = ld16(xp[i] + min(c, p.width - 8));
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int t = 0; t < NT; ++t) a[k][t] = ld16(ap + ((int64_t)step * tiles16 + min(t, most)) * 1024 + 512 * k);
    wave_sync();
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) stage[(8 * i + r8) * 8 + (c8 ^ r8)] = x[i];
    if (64 * step + 64 > p.width && c >= p.width)
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) stage[(8 * i + r8) * 8 + (c8 ^ r8)] = u32x4_t{};
    wave_sync();
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const bf16x8_t f = as_bf16x8(stage[(16 * m + l16) * 8 + ((4 * k + g) ^ (l16 & 7))]);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t * MT + m] = mfma_bf16_16x16x32(as_bf16x8(a[k][t]), f, acc[t * MT + m]);
      }
  }
  // tile i is added up and written by wavefront i % W
  constexpr int KEPT = (T + W - 1) / W;
  const float scale = p.scales ? p.scales[adapter] : 1.f;
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    const int tiles = T - k * W < W ? T - k * W : W;  // the tiles of this turn
    __syncthreads();
#pragma unroll
    for (int i = 0; i < tiles; ++i) sums[wave * TURN + i][lane] = __builtin_bit_cast(u32x4_t, acc[k * W + i]);
    __syncthreads();
    if (wave >= tiles) continue;
    f32x4_t all = __builtin_bit_cast(f32x4_t, sums[wave][lane]);
#pragma unroll
    for (int w = 1; w < W; ++w) all += __builtin_bit_cast(f32x4_t, sums[w * TURN + wave][lane]);
    const int i = k * W + wave, m = i % MT, r = rank0 + 16 * (i / MT) + 4 * g;
    if (16 * m + l16 >= count || r >= p.ranks) continue;
    all *= scale;
    if (p.rank < p.ranks)  // ranks that the adapters do not have, whatever x holds
#pragma unroll
      for (int j = 0; j < 4; ++j) all[j] = r + j < p.rank ? all[j] : 0.f;
    const u32x2_t hi = {pack_bf2(all[0], all[1]), pack_bf2(all[2], all[3])};
    const u32x2_t lo = {pack_bf2(rest(all[0], hi[0] << 16), rest(all[1], hi[0] & 0xffff0000u)),
                        pack_bf2(rest(all[2], hi[1] << 16), rest(all[3], hi[1] & 0xffff0000u))};
    const int64_t row = LISTED ? 16 * m + l16 : row0 + list[16 * m + l16];
    uint16_t *to = h + (row * p.ranks + (r & ~7)) * 2 + (r & 4);
    *reinterpret_cast<u32x2_t *>(to) = hi;
    *reinterpret_cast<u32x2_t *>(to + 8) = lo;
  }
}

// grid: shares x rank groups x blocks of 16 MT rows; a workgroup takes every `shares`-th adapter of its block
template <int MT, int NT>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(AdapterCall p, int groups) {
  // sums of the wavefronts, a kilobyte a tile; before that 2 MT of them as each wavefront's part for x
  constexpr int TURN = MT * NT < kShrinkWaves ? MT * NT : kShrinkWaves;
  __shared__ u32x4_t sums[kShrinkWaves * (TURN > 2 * MT ? TURN : 2 * MT)][64];
  __shared__ int lists[kShrinkWaves][kListRows];
  int at = blockIdx.x;
  const int share = at % p.shares;
  at /= p.shares;
  const int rank0 = at % groups * (16 * NT), row0 = at / groups * (16 * MT);
  int *list = lists[threadIdx.x >> 6];
  const int mine = adapter_of(p, row0, 16 * MT);
  uint64_t left = __ballot(mine >= 0);
  for (int n = 0; left; ++n) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    if (n % p.shares != share) continue;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (MT > 1 && count > 16) {
      if (MT > 2 && count > 32) shrink_rows<MT, NT, false>(p, row0, list, count, adapter, rank0, sums, p.h);
      else shrink_rows<(MT > 1 ? 2 : 1), NT, false>(p, row0, list, count, adapter, rank0, sums, p.h);
    } else {
      shrink_rows<1, NT, false>(p, row0, list, count, adapter, rank0, sums, p.h);
    }
  }
}

// Four k-values a lane: A[m = l % 16][k = 4 (l / 16) + j], B[k][n] alike
__device__ __forceinline__ f32x4_t mfma_bf16_16x16x16(u32x2_t a, u32x2_t b, f32x4_t c) {
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c, 0, 0, 0);
}

// A wavefront's 16 x 64 tile in LDS on its way from columns to rows
constexpr int kTurnRow = 68, kTurn = 16 * kTurnRow;

// out = y + B h of the rows of one adapter in a block, a wavefront's 64 of each STEP columns of the workgroup's span.
// C[column][row] tiles whose columns are ordered so that a pair of tiles gives a lane eight neighbours: row m of tile t is
// column 32 (t / 2) + 8 (m / 4) + 4 (t % 2) + m % 4. They turn in LDS so that y and out are read and written in runs of 128
// bytes of a row, eight rows at a time: 833 MB take 150 us that way, and 197 as 64 bytes of 16 rows, as the tiles lie.
// KS: the ranks in 32s, kept as operands over the columns; 0: 16 ranks; -1: any number of 32s, read again for each 64 columns.
// STEP: the columns of the workgroup's wavefronts.
template <int MT, int KS, int STEP, bool LISTED>
__device__ __forceinline__ void expand_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int col0,
                                            int col_end, float *turn, const uint16_t *h) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, r8 = lane >> 3, c8 = lane & 7;
  const uint16_t *hp[MT];
  int64_t row[2 * MT];  // the lane's rows of y and out: 8 i + r8 of the list
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) row[i] = row0 + list[8 * i + r8];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    hp[m] = h + (LISTED ? 16 * m + l16 : (int64_t)row0 + list[16 * m + l16]) * p.ranks * 2 +
            (KS ? 16 * g : 16 * (g / 2) + 4 * (g % 2));
  }
  constexpr int KEPT = KS > 0 ? KS : 1;
  u32x4_t hi[KEPT][MT], lo[KEPT][MT];  // 16 ranks: the first halves
  auto load_h = [&](int i, int k) __device__ {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (KS == 0) {
        const u32x2_t a = *reinterpret_cast<const u32x2_t *>(hp[m]), b = *reinterpret_cast<const u32x2_t *>(hp[m] + 8);
        hi[i][m] = u32x4_t{a[0], a[1], 0, 0};
        lo[i][m] = u32x4_t{b[0], b[1], 0, 0};
      } else {
        hi[i][m] = ld16(hp[m] + 64 * k);
        lo[i][m] = ld16(hp[m] + 64 * k + 8);
      }
    }
  };
  if constexpr (KS >= 0) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k) load_h(k, k);
  }
  const int ks = KS < 0 ? p.ranks / 32 : KEPT, pairs = (p.out_width + 31) / 32, piece = KS ? 1024 : 512;
  const uint16_t *up = p.up + (int64_t)adapter * pairs * ks * piece + lane * 8;
  for (; col0 < col_end; col0 += STEP) {
    const int c = col0 + 8 * c8;
    u32x4_t y[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) y[i] = c < p.out_width && 8 * i + r8 < count ? ld16(p.y + row[i] * p.y_row + c) : u32x4_t{};
    f32x4_t acc[4][MT] = {};
    auto products = [&](int i, int k) __device__ {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // columns behind the last read the last pair again and are not stored
        const uint16_t *b = up + ((int64_t)min(col0 / 32 + t, pairs - 1) * ks + k) * piece;
        if constexpr (KS == 0) {
          const u32x4_t both = ld16(b);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const u32x2_t f = {both[2 * half], both[2 * half + 1]};
              f32x4_t &c = acc[2 * t + half][m];
              c = mfma_bf16_16x16x16(f, u32x2_t{hi[i][m][0], hi[i][m][1]}, c);
              c = mfma_bf16_16x16x16(f, u32x2_t{lo[i][m][0], lo[i][m][1]}, c);
            }
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bf16x8_t f = as_bf16x8(ld16(b + 512 * half));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              f32x4_t &c = acc[2 * t + half][m];
              c = mfma_bf16_16x16x32(f, as_bf16x8(hi[i][m]), c);
              c = mfma_bf16_16x16x32(f, as_bf16x8(lo[i][m]), c);
            }
          }
        }
      }
    };
    if constexpr (KS >= 0) {
#pragma unroll
      for (int k = 0; k < KEPT; ++k) products(k, k);
    } else {
      for (int k = 0; k < ks; ++k) {
        load_h(0, k);
        products(0, k);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float *tile = turn + (m & 1) * kTurn;
      wave_sync();
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *reinterpret_cast<f32x4_t *>(tile + l16 * kTurnRow + 32 * (t / 2) + 8 * g + 4 * (t % 2)) = acc[t][m];
      wave_sync();
#pragma unroll
      for (int i = 2 * m; i < 2 * m + 2; ++i) {
        const f32x4_t *d = reinterpret_cast<const f32x4_t *>(tile + (8 * (i & 1) + r8) * kTurnRow + 8 * c8);
        const f32x4_t d0 = d[0], d1 = d[1];
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x0 = j < 2 ? d0[2 * j] : d1[2 * j - 4], x1 = j < 2 ? d0[2 * j + 1] : d1[2 * j - 3];
          o[j] = pack_bf2(__uint_as_float(y[i][j] << 16) + x0, __uint_as_float(y[i][j] & 0xffff0000u) + x1);
        }
        if (c < p.out_width && 8 * i + r8 < count) st16(p.out + row[i] * p.out_row + c, o);
      }
    }
  }
}

// Rows without an adapter: y as it is, a wavefront's 64 of each STEP columns, eight of each 8 `shares` rows.
template <int STEP>
__device__ __forceinline__ void copy_rows(const AdapterCall &p, int row0, uint64_t rows, int *list, int share, int shares, int col0,
                                          int col_end) {
  if (rows == 0) return;
  list_rows(rows, list);
  const int lane = threadIdx.x & 63, count = __popcll(rows);
  for (int i = share * 8 + (lane >> 3); i < count; i += 8 * shares) {
    const int64_t row = row0 + list[i];
    for (int c = col0 + 8 * (lane & 7); c < col_end; c += STEP) st16(p.out + row * p.out_row + c, ld16(p.y + row * p.y_row + c));
  }
}

// grid: spans of columns x shares x blocks; a workgroup takes every `shares`-th adapter of its block
template <int KS>
__global__ __launch_bounds__(256, 3) void adapter_expand_kernel(AdapterCall p, int spans, int span, int shares) {
  __shared__ int lists[4][kListRows];
  __shared__ __attribute__((aligned(16))) float turns[4][2 * kTurn];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int at = blockIdx.x;
  const int first = at % spans * span, col0 = first + 64 * wave, col_end = min(first + span, p.out_width);
  at /= spans;
  const int share = at % shares, row0 = at / shares * kExpandRows;
  if (col0 >= col_end) return;
  int *list = lists[wave];
  const int mine = adapter_of(p, row0, kExpandRows);
  uint64_t left = __ballot(mine >= 0);
  if (p.copy)
    copy_rows<256>(p, row0, __ballot(mine < 0 && lane < kExpandRows && row0 + lane < p.rows), list, share, shares, col0, col_end);
  for (int n = 0; left; ++n) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    if (n % shares != share) continue;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (count <= 16) expand_rows<1, KS, 256, false>(p, row0, list, count, adapter, col0, col_end, turns[wave], p.h);
    else expand_rows<kExpandRows / 16, KS, 256, false>(p, row0, list, count, adapter, col0, col_end, turns[wave], p.h);
  }
}

// Both products in one launch for few rows: every workgroup of a span of columns makes s A x of its adapters' rows anew, in LDS.
// Spans of 512 columns or more, as many workgroups as one round of the CUs: one row x 5,120 -> 15,360 of rank 16 takes 6.0 us
// (two launches 7.7, and 4 us more of the host's), 64 rows of 16 adapters 11.1 in spans of 1,024 (512 16.7, 2,048 12.6, two
// launches 13.9). Where it is taken: one_launch.
template <int NT, int KS>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_few_rows_kernel(AdapterCall p, int spans, int span) {
  constexpr int STEP = 64 * kShrinkWaves;
  __shared__ u32x4_t sums[(kShrinkWaves * 2 * kTurn + 255) / 256][64];
  __shared__ __attribute__((aligned(16))) uint16_t h[kFewRows * 16 * NT * 2];
  __shared__ int lists[kShrinkWaves][kListRows];
  static_assert(sizeof(sums) >= kShrinkWaves * 8 * 1024, "the tiles turn where x and the sums were");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = (int)blockIdx.x % spans * span, share = (int)blockIdx.x / spans;
  const int col0 = first + 64 * wave, col_end = min(first + span, p.out_width);
  int *list = lists[wave];
  float *turn = reinterpret_cast<float *>(sums) + wave * 2 * kTurn;
  const int mine = adapter_of(p, 0, kFewRows);
  uint64_t left = __ballot(mine >= 0);
  if (p.copy) copy_rows<STEP>(p, 0, __ballot(mine < 0 && lane < p.rows), list, share, p.shares, col0, col_end);
  for (int n = 0; left; ++n) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    if (n % p.shares != share) continue;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (count <= 16) shrink_rows<1, NT, true>(p, 0, list, count, adapter, 0, sums, h);
    else if (count <= 32) shrink_rows<2, NT, true>(p, 0, list, count, adapter, 0, sums, h);
    else shrink_rows<4, NT, true>(p, 0, list, count, adapter, 0, sums, h);
    __syncthreads();
    if (count <= 16) {
      expand_rows<1, KS, STEP, true>(p, 0, list, count, adapter, col0, col_end, turn, h);
    } else {
      for (int i = 0; i < count; i += 32)
        expand_rows<2, KS, STEP, true>(p, 0, list + i, count - i, adapter, col0, col_end, turn, h + (int64_t)i * p.ranks * 2);
    }
  }
}

// The ranks that are kept: 16, or a multiple of 32; zeros behind the adapter's own.
int kept_ranks(int rank) { return rank <= 16 ? 16 : (rank + 31) / 32 * 32; }

// Whether the one launch for few rows is the faster form. Its workgroups, a span of columns and every `shares`-th registered
// adapter each, make A x anew, so it loses where many rows of wide x fall to few adapters; the host knows the registered ones,
// not those that rows name. Kernel times in us, one launch / two (which are 4 us more of the host's), for rows x width -> columns
// of rank 32: one adapter 16 x 5,120 -> 5,120 7.2 / 8.9, 32 9.2 / 9.5, 48 13.8 / 9.6, 64 15.5 / 9.7; 16 x 13,824 -> 5,120
// 15.9 / 16.8, 24 20.0 / 17.2; 64 x 1,024 -> 1,024 8.2 / 7.0; of four adapters 64 x 5,120 -> 5,120 9.8 / 9.3 with rows of each,
// 14.8 / 9.6 if all name one; of 16 64 x 5,120 -> 15,360 12.9 / 15.2 and 20.3 / 11.8.
constexpr int kFewRowsAlways = 16;
constexpr int64_t kFewChannels = 32 * 5120;
bool one_launch(int64_t rows, int64_t width, int64_t adapters) {
  return rows <= kFewRowsAlways || rows * width <= kFewChannels * std::min(rows, adapters);
}

// Rows of a shrinking workgroup: 16 until there are workgroups enough without, since A is read for each (3,939 rows of rank 32:
// 15.2 us with 16, 21 with 32, 35 with 64; 9,000 of rank 128: 59 with 16, 48 with 32; 40,688 of rank 64, both products: 336, 307,
// 304, and 760, 583, 531 with adapters that change from row to row).
constexpr int kRows32 = 8192, kRows64 = 16384;
// Adapters of a block go to workgroups of their own, and its columns, until there are about this many: 64 rows of 16 adapters x
// 15,360 columns 6.3 us (all adapters in one workgroup 98, in 16 8.1), 256 of them 13.7 (18, 15); 40,688 rows x 5,120 columns,
// both products, 304 us in six spans, 313 in three; 9,000 x 15,360 111 and 125.
constexpr int kShrinkGroups = 512, kExpandShares = 1024, kExpandGroups = 8192;
constexpr int kMostWidth = 1 << 30;  // the kernels step over columns in 32 bits

struct AdapterCut {
  int ranks, row_tiles, rank_tiles, groups, shares, span, expand_shares;
  int64_t shrink, expand;  // workgroups
};
// In 64 bits: rows are any 32-bit number
AdapterCut adapter_cut(int64_t rows, int64_t out_width, int adapters, int rank) {
  AdapterCut c;
  c.ranks = kept_ranks(rank);
  c.row_tiles = rows >= kRows64 ? 4 : rows >= kRows32 ? 2 : 1;
  const int most = c.row_tiles == 4 ? 4 : 8;
  c.rank_tiles = 1;
  while (c.rank_tiles < most && 16 * c.rank_tiles < c.ranks) c.rank_tiles *= 2;
  c.groups = (c.ranks + 16 * c.rank_tiles - 1) / (16 * c.rank_tiles);
  const int64_t blocks = (rows + 16 * c.row_tiles - 1) / (16 * c.row_tiles), of = std::min<int64_t>(rows, adapters);
  c.shares = (int)std::max<int64_t>(1, std::min({of, (int64_t)16 * c.row_tiles, kShrinkGroups / (blocks * c.groups)}));
  c.shrink = blocks * c.groups * c.shares;
  // columns of an expanding workgroup: fewer than all where that leaves too few workgroups
  const int64_t tall = (rows + kExpandRows - 1) / kExpandRows, column_tiles = (out_width + 255) / 256;
  c.expand_shares = (int)std::max<int64_t>(1, std::min({of, (int64_t)16, kExpandShares / (tall * column_tiles)}));
  const int64_t spans = std::min(column_tiles, std::max<int64_t>(1, kExpandGroups / (tall * c.expand_shares)));
  c.span = (int)((column_tiles + spans - 1) / spans) * 256;
  c.expand = tall * c.expand_shares * ((out_width + c.span - 1) / c.span);
  return c;
}

int check_adapter_rows(const void *p, int64_t row, int width, const char *name, bool read) {
  VDNH3_HOST_CHECK(p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && row >= (read ? 0 : width),
                   VDNH3_ERR_INVALID, "adapter_add: %s must be 16-byte aligned with a row stride of a multiple of 8, rows of out "
                   "apart", name);
  return VDNH3_OK;
}

}  // namespace
}  // namespace vdnh3

extern "C" size_t vdnh3_adapter_workspace_bytes(int rows, int rank) {
  if (rows <= 0 || rank <= 0 || rank > 1024) return 0;
  if (rows <= vdnh3::kFewRows && rank <= vdnh3::kFewRanks) return 0;
  return (size_t)rows * vdnh3::kept_ranks(rank) * 4;
}

extern "C" size_t vdnh3_adapter_workspace_wanted(int rows, int width, int adapters, int rank) {
  if (rows <= 0 || width <= 0 || adapters <= 0 || rank <= 0 || rank > 1024) return 0;
  const size_t needed = vdnh3_adapter_workspace_bytes(rows, rank);
  if (needed || vdnh3::one_launch(rows, width, adapters)) return needed;
  return (size_t)rows * vdnh3::kept_ranks(rank) * 4;
}

extern "C" int vdnh3_adapter_add(const uint16_t *y, int64_t y_row, const uint16_t *x, int64_t x_row, const uint16_t *down,
                                 const uint16_t *up, const float *scales, const int32_t *index, uint16_t *out, int64_t out_row,
                                 int rows, int width, int out_width, int adapters, int rank, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  using namespace vdnh3;
  VDNH3_HOST_CHECK(rows > 0 && width > 0 && out_width > 0 && adapters > 0 && rank > 0, VDNH3_ERR_INVALID,
                   "adapter_add: rows, widths, adapters and rank must be positive, got %d rows, %d -> %d, %d of rank %d", rows,
                   width, out_width, adapters, rank);
  VDNH3_HOST_CHECK(width % 8 == 0 && out_width % 8 == 0 && width <= kMostWidth && out_width <= kMostWidth && rank <= 1024,
                   VDNH3_ERR_INVALID, "adapter_add: widths must be multiples of 8, at most 2^30, and the rank at most 1024, got "
                   "%d -> %d, rank %d", width, out_width, rank);
  VDNH3_HOST_CHECK(index != nullptr, VDNH3_ERR_INVALID, "adapter_add: an index is needed");
  if (rows == 1) y_row = out_row = out_width, x_row = width;  // one row has no stride, whatever a caller passes for it
  int rc = check_adapter_rows(x, x_row, width, "x", true);
  if (!rc) rc = check_adapter_rows(y, y_row, out_width, "y", true);
  if (!rc) rc = check_adapter_rows(out, out_row, out_width, "out", false);
  if (rc) return rc;
  VDNH3_HOST_CHECK(down && up && reinterpret_cast<uintptr_t>(down) % 16 == 0 && reinterpret_cast<uintptr_t>(up) % 16 == 0,
                   VDNH3_ERR_INVALID, "adapter_add: down and up must be 16-byte aligned");
  VDNH3_HOST_CHECK(out != y || out_row == y_row, VDNH3_ERR_INVALID, "adapter_add: out over y needs y's row stride");
  const size_t needed = vdnh3_adapter_workspace_bytes(rows, rank);
  VDNH3_HOST_CHECK(needed == 0 ||
                       (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= needed),
                   VDNH3_ERR_INVALID, "adapter_add: needs a 16-byte aligned workspace of %zu bytes", needed);
  const AdapterCut c = adapter_cut(rows, out_width, adapters, rank);
  rc = check_grid(c.shrink, 64 * kShrinkWaves, "adapter_add");
  if (!rc) rc = check_grid(c.expand, 256, "adapter_add");
  if (rc) return rc;
  AdapterCall p{x, y, down, up, out, x_row, y_row, out_row, scales, index, static_cast<uint16_t *>(workspace), rows, width,
                out_width, adapters, rank, c.ranks, c.shares, out != y};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t wanted = vdnh3_adapter_workspace_wanted(rows, width, adapters, rank);
  const bool room = workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= wanted;
  if (needed == 0 && (wanted == 0 || !room)) {
    p.shares = std::min({rows, adapters, 16});
    const int wide = (out_width + 511) / 512, span = 512 * ((wide * p.shares + 255) / 256), spans = (out_width + span - 1) / span;
    auto few = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(spans * p.shares), dim3(64 * kShrinkWaves), 0, s, p, spans, span);
    };
    if (c.ranks == 16) few(adapter_few_rows_kernel<1, 0>);
    else if (c.ranks == 32) few(adapter_few_rows_kernel<2, 1>);
    else few(adapter_few_rows_kernel<4, 2>);
    return check_launch("adapter_add");
  }
  auto shrink = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)c.shrink), dim3(64 * kShrinkWaves), 0, s, p, c.groups);
  };
  auto by_ranks = [&](auto rows16) {
    constexpr int MT = decltype(rows16)::value;
    if (c.rank_tiles == 1) shrink(adapter_shrink_kernel<MT, 1>);
    else if (c.rank_tiles == 2) shrink(adapter_shrink_kernel<MT, 2>);
    else if (c.rank_tiles == 4) shrink(adapter_shrink_kernel<MT, 4>);
    else if constexpr (MT < 4) shrink(adapter_shrink_kernel<MT, 8>);
  };
  if (c.row_tiles == 4) by_ranks(std::integral_constant<int, 4>());
  else if (c.row_tiles == 2) by_ranks(std::integral_constant<int, 2>());
  else by_ranks(std::integral_constant<int, 1>());
  rc = check_launch("adapter_add");
  if (rc) return rc;
  const int spans = (out_width + c.span - 1) / c.span;
  auto expand = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)c.expand), dim3(256), 0, s, p, spans, c.span, c.expand_shares);
  };
  if (c.ranks == 16) expand(adapter_expand_kernel<0>);
  else if (c.ranks == 32) expand(adapter_expand_kernel<1>);
  else if (c.ranks == 64) expand(adapter_expand_kernel<2>);
  else expand(adapter_expand_kernel<-1>);
  return check_launch("adapter_add");
}
