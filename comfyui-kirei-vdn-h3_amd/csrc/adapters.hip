// Low-rank adapters of many requests beside a shared projection on gfx950, bf16:
//
//   out_t = bf16(y_t + s_i B_i (A_i x_t)),  i = index[t]     A_i: [rank, width], B_i: [out_width, rank], s_i fp32
//
// y is the projection's output for all rows; a row whose index names no adapter keeps it. h = A x is held in fp32, summed over
// the parts of the width that different workgroups take; s h meets B as two bf16 numbers (16 bits of it), and the sum with y is
// rounded once. Rows are taken in blocks of 64 neighbours; a block finds the adapters in it by ballots and takes their rows
// together, so the rows of one request share each fragment of its adapter, in whatever order requests lie.
#include <algorithm>

#include "common.h"

namespace vdnh3 {
namespace {

constexpr int kBlockRows = 64;  // of an expanding workgroup; the most that a list holds
constexpr int kShrinkWaves = 8;

struct AdapterCall {
  const uint16_t *x, *y, *down, *up;
  uint16_t *out;
  int64_t x_row, y_row, out_row;
  const float *scales;
  const int32_t *index;
  uint16_t *h;  // [rows, rank rounded up to 32 in eights, 2, 8]: s A x as two bf16 numbers
  int rows, width, out_width, adapters, rank, rank32, shares, copy;
};

// The adapter of each of a block's rows, a lane a row: -1 for none and behind the last row.
__device__ __forceinline__ int adapter_of(const AdapterCall &p, int row0, int block_rows) {
  const int lane = threadIdx.x & 63;
  const int i = lane < block_rows && row0 + lane < p.rows ? p.index[row0 + lane] : -1;
  return i >= 0 && i < p.adapters ? i : -1;
}

// The rows of `mask`, one behind another, as a wavefront's list; the last one repeats behind its end.
__device__ __forceinline__ void list_rows(uint64_t mask, int *list) {
  const int lane = threadIdx.x & 63, at = __popcll(mask & ((1ull << lane) - 1)), count = __popcll(mask);
  if ((mask >> lane) & 1) list[at] = lane;
  if (lane >= count) list[lane] = 63 - __builtin_clzll(mask);
}

// s A x of the rows of one adapter in a block: the wavefronts take steps of 64 channels in turn and add their sums up in LDS.
// C[rank][row] tiles: a lane has four ranks of a row.
template <int MT, int NT>
__device__ __forceinline__ void shrink_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int rank0,
                                            f32x4_t (*sums)[64]) {
  constexpr int T = MT * NT, W = kShrinkWaves;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const uint16_t *xp[MT], *ap[NT];
  bool has[NT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xp[m] = p.x + (int64_t)(row0 + list[16 * m + l16]) * p.x_row;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = rank0 + 16 * t + l16;
    has[t] = r < p.rank;
    ap[t] = p.down + ((int64_t)adapter * p.rank + (has[t] ? r : 0)) * p.width;
  }
  f32x4_t acc[T] = {};
  auto products = [&](const u32x4_t *a, const u32x4_t *x) __device__ {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[t * MT + m] = mfma_bf16_16x16x32(as_bf16x8(a[t]), as_bf16x8(x[m]), acc[t * MT + m]);
  };
  int c0 = 64 * wave;
  for (; c0 + 64 <= p.width; c0 += 64 * W) {
    u32x4_t a[2][NT], x[2][MT];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = c0 + 32 * k + 8 * g;
#pragma unroll
      for (int m = 0; m < MT; ++m) x[k][m] = ld16(xp[m] + c);
#pragma unroll
      for (int t = 0; t < NT; ++t) a[k][t] = has[t] ? ld16(ap[t] + c) : u32x4_t{};
    }
    products(a[0], x[0]);
    products(a[1], x[1]);
  }
  for (int c1 = c0; c1 < p.width && c1 < c0 + 64; c1 += 32) {
    const int c = c1 + 8 * g;
    const bool in = c < p.width;
    u32x4_t a[NT], x[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) a[t] = in && has[t] ? ld16(ap[t] + c) : u32x4_t{};
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = in ? ld16(xp[m] + c) : u32x4_t{};
    products(a, x);
  }
  // tile i is added up and written by wavefront i % W
  constexpr int KEPT = (T + W - 1) / W;
  const float scale = p.scales ? p.scales[adapter] : 1.f;
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    const int tiles = T - k * W < W ? T - k * W : W;  // the tiles of this turn
    __syncthreads();
#pragma unroll
    for (int i = 0; i < tiles; ++i) sums[wave * W + i][lane] = acc[k * W + i];
    __syncthreads();
    if (wave >= tiles) continue;
    f32x4_t all = sums[wave][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) all += sums[w * W + wave][lane];
    const int i = k * W + wave, m = i % MT, r = rank0 + 16 * (i / MT) + 4 * g;
    if (16 * m + l16 >= count || r >= p.rank32) continue;
    all *= scale;
    const u32x2_t hi = {pack_bf2(all[0], all[1]), pack_bf2(all[2], all[3])};
    const u32x2_t lo = {pack_bf2(all[0] - __uint_as_float(hi[0] << 16), all[1] - __uint_as_float(hi[0] & 0xffff0000u)),
                        pack_bf2(all[2] - __uint_as_float(hi[1] << 16), all[3] - __uint_as_float(hi[1] & 0xffff0000u))};
    uint16_t *to = p.h + ((int64_t)(row0 + list[16 * m + l16]) * p.rank32 + (r & ~7)) * 2 + (r & 4);
    *reinterpret_cast<u32x2_t *>(to) = hi;
    *reinterpret_cast<u32x2_t *>(to + 8) = lo;
  }
}

// grid: shares x rank groups x blocks of 16 MT rows; a workgroup takes every `shares`-th adapter of its block
template <int MT, int NT>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(AdapterCall p, int groups) {
  __shared__ f32x4_t sums[kShrinkWaves * kShrinkWaves][64];
  __shared__ int lists[kShrinkWaves][kBlockRows];
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
      if (MT > 2 && count > 32) shrink_rows<MT, NT>(p, row0, list, count, adapter, rank0, sums);
      else shrink_rows<(MT > 1 ? 2 : 1), NT>(p, row0, list, count, adapter, rank0, sums);
    } else {
      shrink_rows<1, NT>(p, row0, list, count, adapter, rank0, sums);
    }
  }
}

// s A x of a row, eight ranks, as the operand's two bf16 numbers
struct HalfPair {
  u32x4_t hi, lo;
};
__device__ __forceinline__ HalfPair load_h(const uint16_t *row, int r) { return HalfPair{ld16(row + 2 * r), ld16(row + 2 * r + 8)}; }

// out = y + s B h of the rows of one adapter in a block, a wavefront's 64 of each 256 columns of the workgroup's span.
// C[column][row] tiles whose columns are ordered so that a pair of tiles gives a lane eight neighbours: row m of tile t is
// column 32 (t / 2) + 8 (m / 4) + 4 (t % 2) + m % 4. KS: the ranks in 32s, kept as operands over the columns; 0: any number of
// them, read again for each 64 columns.
template <int MT, int KS>
__device__ __forceinline__ void expand_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int col0,
                                            int col_end) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint16_t *hp[MT];
  int64_t row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    row[m] = row0 + list[16 * m + l16];
    hp[m] = p.h + row[m] * p.rank32 * 2;
  }
  HalfPair h[KS ? KS : 1][MT];
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int m = 0; m < MT; ++m) h[k][m] = load_h(hp[m], 32 * k + 8 * g);
  const uint16_t *up = p.up + (int64_t)adapter * p.out_width * p.rank;
  for (; col0 < col_end; col0 += 256) {
    u32x4_t y[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int c = col0 + 32 * t + 8 * g;
        y[m][t] = c < p.out_width && 16 * m + l16 < count ? ld16(p.y + row[m] * p.y_row + c) : u32x4_t{};
      }
    f32x4_t acc[4][MT] = {};
    auto products = [&](int r0, const HalfPair *hk) __device__ {
      const int r = r0 + 8 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int c = col0 + 32 * (t / 2) + 8 * (l16 / 4) + 4 * (t % 2) + l16 % 4;
        const u32x4_t b = r < p.rank && c < p.out_width ? ld16(up + (int64_t)c * p.rank + r) : u32x4_t{};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[t][m] = mfma_bf16_16x16x32(as_bf16x8(b), as_bf16x8(hk[m].hi), acc[t][m]);
          acc[t][m] = mfma_bf16_16x16x32(as_bf16x8(b), as_bf16x8(hk[m].lo), acc[t][m]);
        }
      }
    };
    if constexpr (KS > 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k) products(32 * k, h[k]);
    } else {
      for (int r0 = 0; r0 < p.rank; r0 += 32) {
#pragma unroll
        for (int m = 0; m < MT; ++m) h[0][m] = load_h(hp[m], r0 + 8 * g);
        products(r0, h[0]);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (16 * m + l16 >= count) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int c = col0 + 32 * t + 8 * g;
        if (c >= p.out_width) continue;
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4_t &d = acc[2 * t + j / 2][m];
          o[j] = pack_bf2(__uint_as_float(y[m][t][j] << 16) + d[2 * (j % 2)],
                          __uint_as_float(y[m][t][j] & 0xffff0000u) + d[2 * (j % 2) + 1]);
        }
        st16(p.out + row[m] * p.out_row + c, o);
      }
    }
  }
}

// grid: spans of columns x shares x blocks; a workgroup takes every `shares`-th adapter of its block
template <int KS>
__global__ __launch_bounds__(256) void adapter_expand_kernel(AdapterCall p, int spans, int span, int shares) {
  __shared__ int lists[4][kBlockRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int at = blockIdx.x;
  const int first = at % spans * span, col0 = first + 64 * wave, col_end = min(first + span, p.out_width);
  at /= spans;
  const int share = at % shares, row0 = at / shares * kBlockRows;
  if (col0 >= col_end) return;
  int *list = lists[wave];
  const int mine = adapter_of(p, row0, kBlockRows);
  uint64_t left = __ballot(mine >= 0);
  if (p.copy) {  // rows without an adapter: y as it is
    const uint64_t none = __ballot(mine < 0 && row0 + lane < p.rows);
    if (none) {
      list_rows(none, list);
      const int count = __popcll(none);
      for (int i = share * 8 + (lane >> 3); i < count; i += 8 * shares) {
        const int64_t row = row0 + list[i];
        for (int c = col0 + 8 * (lane & 7); c < col_end; c += 256) st16(p.out + row * p.out_row + c, ld16(p.y + row * p.y_row + c));
      }
    }
  }
  for (int n = 0; left; ++n) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    if (n % shares != share) continue;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (count <= 16) expand_rows<1, KS>(p, row0, list, count, adapter, col0, col_end);
    else if (count <= 32) expand_rows<2, KS>(p, row0, list, count, adapter, col0, col_end);
    else expand_rows<4, KS>(p, row0, list, count, adapter, col0, col_end);
  }
}

#ifndef ROWS64
#define ROWS64 16384
#endif
#ifndef ROWS32
#define ROWS32 8192
#endif
#ifndef EX_WG
#define EX_WG 2048
#endif
struct AdapterCut {
  int rank32, row_tiles, rank_tiles, groups, shares, span, expand_shares;
  int64_t shrink, expand;  // workgroups
};
AdapterCut adapter_cut(int rows, int out_width, int adapters, int rank) {
  AdapterCut c;
  c.rank32 = (rank + 31) / 32 * 32;
  c.row_tiles = rows >= ROWS64 ? 4 : rows >= ROWS32 ? 2 : 1;
  const int most = c.row_tiles == 4 ? 4 : 8;
  c.rank_tiles = 2;
  while (c.rank_tiles < most && 16 * c.rank_tiles < c.rank32) c.rank_tiles *= 2;
  c.groups = (c.rank32 + 16 * c.rank_tiles - 1) / (16 * c.rank_tiles);
  const int64_t blocks = (rows + 16 * c.row_tiles - 1) / (16 * c.row_tiles), of = std::min(rows, adapters);
  c.shares = (int)std::max<int64_t>(1, std::min({of, (int64_t)16 * c.row_tiles, 512 / (blocks * c.groups)}));
  c.shrink = blocks * c.groups * c.shares;
  // columns of an expanding workgroup: fewer than all where that leaves too few workgroups
  const int64_t tall = (rows + kBlockRows - 1) / kBlockRows, column_tiles = (out_width + 255) / 256;
  c.expand_shares = (int)std::max<int64_t>(1, std::min({of, (int64_t)16, EX_WG / (tall * column_tiles)}));
  const int64_t spans = std::min(column_tiles, std::max<int64_t>(1, EX_WG / (tall * c.expand_shares)));
  c.span = (int)((column_tiles + spans - 1) / spans) * 256;
  c.expand = tall * c.expand_shares * ((out_width + c.span - 1) / c.span);
  return c;
}

int check_adapter_rows(const void *p, int64_t row, int width, const char *name, bool read) {
  VDNH3_HOST_CHECK(p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && (row >= width || (read && row == 0)),
                   VDNH3_ERR_INVALID, "adapter_add: %s must be 16-byte aligned with a row stride of a multiple of 8 that covers "
                   "the width", name);
  return VDNH3_OK;
}

}  // namespace
}  // namespace vdnh3

extern "C" size_t vdnh3_adapter_workspace_bytes(int rows, int rank) {
  if (rows <= 0 || rank <= 0 || rank > 1024) return 0;
  return (size_t)rows * ((rank + 31) / 32 * 32) * 4;
}

extern "C" int vdnh3_adapter_add(const uint16_t *y, int64_t y_row, const uint16_t *x, int64_t x_row, const uint16_t *down,
                                 const uint16_t *up, const float *scales, const int32_t *index, uint16_t *out, int64_t out_row,
                                 int rows, int width, int out_width, int adapters, int rank, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  using namespace vdnh3;
  VDNH3_HOST_CHECK(rows > 0 && width > 0 && out_width > 0 && adapters > 0 && rank > 0, VDNH3_ERR_INVALID,
                   "adapter_add: rows, widths, adapters and rank must be positive, got %d rows, %d -> %d, %d of rank %d", rows, width,
                   out_width, adapters, rank);
  VDNH3_HOST_CHECK(width % 8 == 0 && out_width % 8 == 0 && rank % 8 == 0 && rank <= 1024, VDNH3_ERR_INVALID,
                   "adapter_add: widths and rank must be multiples of 8, the rank at most 1024, got %d -> %d, rank %d", width,
                   out_width, rank);
  VDNH3_HOST_CHECK(index != nullptr, VDNH3_ERR_INVALID, "adapter_add: an index is needed");
  if (rows == 1) y_row = out_row = out_width, x_row = width;  // one row has no stride, whatever a caller passes for it
  int rc = check_adapter_rows(x, x_row, width, "x", true);
  if (!rc) rc = check_adapter_rows(y, y_row, out_width, "y", true);
  if (!rc) rc = check_adapter_rows(out, out_row, out_width, "out", false);
  if (!rc) rc = check_adapter_rows(down, width, width, "down", true);
  if (!rc) rc = check_adapter_rows(up, rank, rank, "up", true);
  if (rc) return rc;
  VDNH3_HOST_CHECK(out != y || out_row == y_row, VDNH3_ERR_INVALID, "adapter_add: out over y needs y's row stride");
  const size_t needed = vdnh3_adapter_workspace_bytes(rows, rank);
  VDNH3_HOST_CHECK(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= needed,
                   VDNH3_ERR_INVALID, "adapter_add: needs a 16-byte aligned workspace of %zu bytes", needed);
  const AdapterCut c = adapter_cut(rows, out_width, adapters, rank);
  rc = check_grid(c.shrink, 64 * kShrinkWaves, "adapter_add");
  if (!rc) rc = check_grid(c.expand, 256, "adapter_add");
  if (rc) return rc;
  const AdapterCall p{x, y, down, up, out, x_row, y_row, out_row, scales, index, static_cast<uint16_t *>(workspace), rows, width,
                      out_width, adapters, rank, c.rank32, c.shares, out != y};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto shrink = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)c.shrink), dim3(64 * kShrinkWaves), 0, s, p, c.groups); };
  if (c.row_tiles == 4)
    c.rank_tiles == 2 ? shrink(adapter_shrink_kernel<4, 2>) : shrink(adapter_shrink_kernel<4, 4>);
  else if (c.row_tiles == 2)
    c.rank_tiles == 2 ? shrink(adapter_shrink_kernel<2, 2>) : c.rank_tiles == 4 ? shrink(adapter_shrink_kernel<2, 4>) : shrink(adapter_shrink_kernel<2, 8>);
  else
    c.rank_tiles == 2 ? shrink(adapter_shrink_kernel<1, 2>) : c.rank_tiles == 4 ? shrink(adapter_shrink_kernel<1, 4>) : shrink(adapter_shrink_kernel<1, 8>);
  rc = check_launch("adapter_add");
  if (rc) return rc;
  const int spans = (out_width + c.span - 1) / c.span;
  auto expand = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)c.expand), dim3(256), 0, s, p, spans, c.span, c.expand_shares); };
  rank <= 32 ? expand(adapter_expand_kernel<1>) : rank <= 64 ? expand(adapter_expand_kernel<2>) : expand(adapter_expand_kernel<0>);
  return check_launch("adapter_add");
}
