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

constexpr int kBlockRows = 64;
constexpr int kRankGroup = 128;  // ranks that a shrinking workgroup takes at most

struct AdapterCall {
  const uint16_t *x, *y, *down, *up;
  uint16_t *out;
  int64_t x_row, y_row, out_row;
  const float *scales;
  const int32_t *index;
  float *h;  // [parts, rows, rank rounded up to 16]
  int rows, width, out_width, adapters, rank, rank16, parts, part_width, shares, copy;
};

// The adapter of each of a block's rows, a lane a row: -1 for none and behind the last row.
__device__ __forceinline__ int adapter_of(const AdapterCall &p, int row0) {
  const int r = row0 + ((int)threadIdx.x & 63);
  const int i = r < p.rows ? p.index[r] : -1;
  return i >= 0 && i < p.adapters ? i : -1;
}

// The rows of `mask`, one behind another, as a wavefront's list; the last one repeats behind its end.
__device__ __forceinline__ void list_rows(uint64_t mask, int *list) {
  const int lane = threadIdx.x & 63, at = __popcll(mask & ((1ull << lane) - 1)), count = __popcll(mask);
  if ((mask >> lane) & 1) {
    list[at] = lane;
    if (at == count - 1)
      for (int i = count; i < kBlockRows; ++i) list[i] = lane;
  }
}

// h = A x of one block, adapter and part of the width: four wavefronts, each with a quarter of the part, whose sums meet in LDS.
// C[rank][row] tiles: a lane keeps four ranks of a row.
template <int MT, int NT>
__device__ __forceinline__ void shrink_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int part,
                                            int rank0, f32x4_t (*sums)[4 * NT][64]) {
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
  f32x4_t acc[NT][MT] = {};
  const int begin = part * p.part_width, end = min(begin + p.part_width, p.width);
  for (int c0 = begin + 32 * wave; c0 < end; c0 += 128) {
    const int c = c0 + 8 * g;
    const bool in = c < end;
    u32x4_t a[NT], x[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) a[t] = in && has[t] ? ld16(ap[t] + c) : u32x4_t{};
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = in ? ld16(xp[m] + c) : u32x4_t{};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[t][m] = mfma_bf16_16x16x32(as_bf16x8(a[t]), as_bf16x8(x[m]), acc[t][m]);
  }
  // wavefronts 2 and 3 give their sums to 0 and 1, then 1 to 0
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) sums[wave - half][t * MT + m][lane] = acc[t][m];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] += sums[wave][t * MT + m][lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (16 * m + l16 >= count) continue;
    float *to = p.h + ((int64_t)part * p.rows + row0 + list[16 * m + l16]) * p.rank16 + rank0 + 4 * g;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (rank0 + 16 * t < p.rank16) *reinterpret_cast<f32x4_t *>(to + 16 * t) = acc[t][m];
  }
}

// grid: parts x shares x rank groups x blocks; a workgroup takes every `shares`-th adapter of its block
template <int NT>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(AdapterCall p, int groups) {
  __shared__ f32x4_t sums[2][4 * NT][64];
  __shared__ int lists[4][kBlockRows];
  int at = blockIdx.x;
  const int part = at % p.parts;
  at /= p.parts;
  const int share = at % p.shares;
  at /= p.shares;
  const int rank0 = at % groups * (16 * NT), row0 = at / groups * kBlockRows;
  int *list = lists[threadIdx.x >> 6];
  const int mine = adapter_of(p, row0);
  uint64_t left = __ballot(mine >= 0);
  for (int n = 0; left; ++n) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    if (n % p.shares != share) continue;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (count <= 16) shrink_rows<1, NT>(p, row0, list, count, adapter, part, rank0, sums);
    else if (count <= 32) shrink_rows<2, NT>(p, row0, list, count, adapter, part, rank0, sums);
    else shrink_rows<4, NT>(p, row0, list, count, adapter, part, rank0, sums);
  }
}

// out = y + s B h of a wavefront's 64 columns and the rows of one adapter in a block. C[column][row] tiles whose columns are
// ordered so that a pair of tiles gives a lane eight neighbours: row m of tile t is column 32 (t / 2) + 8 (m / 4) + 4 (t % 2) + m % 4.
template <int MT>
__device__ __forceinline__ void expand_rows(const AdapterCall &p, int row0, const int *list, int count, int adapter, int col0) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  f32x4_t acc[4][MT] = {};
  const float scale = p.scales ? p.scales[adapter] : 1.f;
  for (int r0 = 0; r0 < p.rank; r0 += 32) {
    const int r = r0 + 8 * g;
    u32x4_t hi[MT], lo[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f32x4_t a = {}, b = {};
      if (r < p.rank) {
        const float *from = p.h + (int64_t)(row0 + list[16 * m + l16]) * p.rank16 + r;
        for (int part = 0; part < p.parts; ++part) {
          const f32x4_t *f = reinterpret_cast<const f32x4_t *>(from + (int64_t)part * p.rows * p.rank16);
          a += f[0];
          b += f[1];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x0 = (j < 2 ? a[2 * j] : b[2 * j - 4]) * scale, x1 = (j < 2 ? a[2 * j + 1] : b[2 * j - 3]) * scale;
        hi[m][j] = pack_bf2(x0, x1);
        lo[m][j] = pack_bf2(x0 - __uint_as_float(hi[m][j] << 16), x1 - __uint_as_float(hi[m][j] & 0xffff0000u));
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int c = col0 + 32 * (t / 2) + 8 * (l16 / 4) + 4 * (t % 2) + l16 % 4;
      const u32x4_t b = r < p.rank && c < p.out_width ? ld16(p.up + ((int64_t)adapter * p.out_width + c) * p.rank + r) : u32x4_t{};
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        acc[t][m] = mfma_bf16_16x16x32(as_bf16x8(b), as_bf16x8(hi[m]), acc[t][m]);
        acc[t][m] = mfma_bf16_16x16x32(as_bf16x8(b), as_bf16x8(lo[m]), acc[t][m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (16 * m + l16 >= count) continue;
    const int row = row0 + list[16 * m + l16];
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      const int c = col0 + 16 * t + 8 * g;
      if (c >= p.out_width) continue;
      const u32x4_t y = ld16(p.y + (int64_t)row * p.y_row + c);
      u32x4_t o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4_t &d = acc[t + j / 2][m];
        o[j] = pack_bf2(__uint_as_float(y[j] << 16) + d[2 * (j % 2)], __uint_as_float(y[j] & 0xffff0000u) + d[2 * (j % 2) + 1]);
      }
      st16(p.out + (int64_t)row * p.out_row + c, o);
    }
  }
}

// grid: column tiles of 256 x blocks
__global__ __launch_bounds__(256) void adapter_expand_kernel(AdapterCall p, int column_tiles) {
  __shared__ int lists[4][kBlockRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col0 = (int)blockIdx.x % column_tiles * 256 + 64 * wave, row0 = (int)blockIdx.x / column_tiles * kBlockRows;
  if (col0 >= p.out_width) return;
  int *list = lists[wave];
  const int mine = adapter_of(p, row0);
  uint64_t left = __ballot(mine >= 0);
  if (p.copy) {  // rows without an adapter: y as it is
    const uint64_t none = __ballot(mine < 0 && row0 + lane < p.rows);
    list_rows(none, list);
    const int count = __popcll(none), c = col0 + 8 * (lane & 7);
    for (int i = lane >> 3; i < count; i += 8) {
      const int64_t row = row0 + list[i];
      if (c < p.out_width) st16(p.out + row * p.out_row + c, ld16(p.y + row * p.y_row + c));
    }
  }
  while (left) {
    const int adapter = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t rows = __ballot(mine == adapter);
    left &= ~rows;
    list_rows(rows, list);
    const int count = __popcll(rows);
    if (count <= 16) expand_rows<1>(p, row0, list, count, adapter, col0);
    else if (count <= 32) expand_rows<2>(p, row0, list, count, adapter, col0);
    else expand_rows<4>(p, row0, list, count, adapter, col0);
  }
}

struct AdapterCut {
  int blocks, rank16, tiles, groups, parts, part_width, shares;
};
AdapterCut adapter_cut(int rows, int width, int adapters, int rank) {
  AdapterCut c;
  c.blocks = (rows + kBlockRows - 1) / kBlockRows;
  c.rank16 = (rank + 15) / 16 * 16;
  const int tiles = std::min(c.rank16, kRankGroup) / 16;
  c.tiles = tiles <= 1 ? 1 : tiles <= 2 ? 2 : tiles <= 4 ? 4 : 8;
  c.groups = (c.rank16 + 16 * c.tiles - 1) / (16 * c.tiles);
  c.shares = c.blocks >= 256 ? 1 : std::min(std::min(rows, adapters), 16);
  // parts of the width until the workgroups are two a CU, of 128 channels or more
  const int64_t wanted = 512 / ((int64_t)c.blocks * c.groups * std::min(c.shares, 4)), most = (width + 127) / 128;
  c.parts = (int)std::max<int64_t>(1, std::min(std::min(wanted, most), (int64_t)16));
  c.part_width = ((width + c.parts - 1) / c.parts + 127) / 128 * 128;
  c.parts = (width + c.part_width - 1) / c.part_width;
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

extern "C" size_t vdnh3_adapter_workspace_bytes(int rows, int width, int adapters, int rank) {
  if (rows <= 0 || width <= 0 || adapters <= 0 || rank <= 0) return 0;
  const vdnh3::AdapterCut c = vdnh3::adapter_cut(rows, width, adapters, rank);
  return (size_t)c.parts * rows * c.rank16 * 4;
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
  const AdapterCut c = adapter_cut(rows, width, adapters, rank);
  VDNH3_HOST_CHECK(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                       workspace_bytes >= vdnh3_adapter_workspace_bytes(rows, width, adapters, rank),
                   VDNH3_ERR_INVALID, "adapter_add: needs a 16-byte aligned workspace of %zu bytes",
                   vdnh3_adapter_workspace_bytes(rows, width, adapters, rank));
  const int column_tiles = (out_width + 255) / 256;
  const int64_t shrink = (int64_t)c.blocks * c.groups * c.shares * c.parts, expand = (int64_t)c.blocks * column_tiles;
  rc = check_grid(shrink, 256, "adapter_add");
  if (!rc) rc = check_grid(expand, 256, "adapter_add");
  if (rc) return rc;
  const AdapterCall p{x, y, down, up, out, x_row, y_row, out_row, scales, index, static_cast<float *>(workspace), rows, width,
                      out_width, adapters, rank, c.rank16, c.parts, c.part_width, c.shares, out != y};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)shrink), threads(256);
  if (c.tiles == 1) hipLaunchKernelGGL(adapter_shrink_kernel<1>, grid, threads, 0, s, p, c.groups);
  else if (c.tiles == 2) hipLaunchKernelGGL(adapter_shrink_kernel<2>, grid, threads, 0, s, p, c.groups);
  else if (c.tiles == 4) hipLaunchKernelGGL(adapter_shrink_kernel<4>, grid, threads, 0, s, p, c.groups);
  else hipLaunchKernelGGL(adapter_shrink_kernel<8>, grid, threads, 0, s, p, c.groups);
  rc = check_launch("adapter_add");
  if (rc) return rc;
  hipLaunchKernelGGL(adapter_expand_kernel, dim3((unsigned)expand), threads, 0, s, p, column_tiles);
  return check_launch("adapter_add");
}
