// Around the products with four-bit matrices: rows of bfloat16 as the parts that multiply four-bit entries, the scales of stacked gate and up rows
// regrouped, and the weighted sum of the experts' results.  Kernels and their launches, for the two libraries that have products.
#pragma once
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"

#define MX4_ROWS_THREADS 256

// act(g) * u in 32 bits.  Sums that are not numbers (a row or a block of weights that is not finite) stay so: the limits of two activations would turn
// them into numbers (0, or the limit); the others pass them on (2,048 rows through 64 experts of 2,048 x 1,408: 313 us; asked of all 340, of none 334).
__device__ __forceinline__ float mx4_gated(int activation, float g, float u, float param) {
  if ((activation == SRB_ACT_RELU2 || activation == SRB_ACT_SWIGLU_CLAMP) && (isnan(g) || isnan(u))) return __uint_as_float(0x7fc00000u);
  return srb_gated<true>(activation, g, u, param);
}

template <bool WIDE>
__device__ __forceinline__ void mx4_load_eight(const __nv_bfloat16* __restrict__ src, int left, bool live, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (!live) return;
  if (WIDE && left >= 8) mx4_unpack_bf16(*reinterpret_cast<const uint4*>(src), v);
  else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) v[i] = srb_to_float(src[i]);
  }
}

// Eight entries of 128 of a row (lane of 16) as the two eight-bit parts of mx4.cuh, and the row's scale words.
struct Mx4SplitEight {
  uint2 high, low;
  unsigned high_word, low_word;
};
__device__ __forceinline__ Mx4SplitEight mx4_split_eight(const float (&v)[8], int lane) {
  unsigned most = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned high = mx8_scale_high(most), low = mx8_scale_low(high);
  unsigned h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mx8_split(v[2 * i], v[2 * i + 1], high, low, h[i], l[i]);
  // (the lanes of a block have the same)
  Mx4SplitEight e = {make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16), make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16), high << (8 * (lane >> 2)),
                     low << (8 * (lane >> 2))};
#pragma unroll
  for (int offset = 4; offset <= 8; offset <<= 1) {
    e.high_word |= __shfl_xor_sync(0xffffffffu, e.high_word, offset);
    e.low_word |= __shfl_xor_sync(0xffffffffu, e.low_word, offset);
  }
  return e;
}
// to `dst` and `dst + part`, `word` and `word + scale_part`
__device__ __forceinline__ void mx4_store_split(const Mx4SplitEight& e, int lane, uint8_t* dst, size_t part, uint8_t* word, size_t scale_part) {
  *reinterpret_cast<uint2*>(dst) = e.high;
  *reinterpret_cast<uint2*>(dst + part) = e.low;
  if (lane == 0) {
    *reinterpret_cast<unsigned*>(word) = e.high_word;
    *reinterpret_cast<unsigned*>(word + scale_part) = e.low_word;
  }
}

// Rows of bfloat16 as parts [2, rows, 128 * column tiles] bytes, zero behind a row's last entry, and their scales [2, row tiles, column tiles, 512]
// in the tiles of mx4.cuh (those of rows behind the last are not written: they are read, but only for sums that nobody stores).
template <bool WIDE>
__global__ void __launch_bounds__(MX4_ROWS_THREADS)
mx4_split_kernel(const __nv_bfloat16* __restrict__ x, size_t pitch, int rows, int width, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_ROWS_THREADS / 16) + (threadIdx.x >> 4);
  const int row = (int)(item / k_tiles), kt = (int)(item % k_tiles), k = kt * 128 + lane * 8;
  float v[8];
  mx4_load_eight<WIDE>(x + (size_t)row * pitch + k, width - k, row < rows, v);
  const Mx4SplitEight e = mx4_split_eight(v, lane);
  if (row < rows)
    mx4_store_split(e, lane, parts + ((size_t)row * k_tiles * 128 + k), (size_t)rows * k_tiles * 128, scales + mx4_scale_word(row, kt, k_tiles),
                    (size_t)mx4_tiles(rows) * k_tiles * MX4_TILE_BYTES);
}

// Scales of stacked gate and up rows (2 * inner rows a matrix) in groups: `group` gate rows, the `group` up rows of the same features, room for
// `room` rows (a multiple of 128) a group.  A product tile's scales are whole tiles then, wherever the up rows begin.  Matrices whose
// slots the product does not take are left out.  A thread has the 16 bytes of four rows, 32 apart.
struct Mx4GatedScales {
  const unsigned* scales;
  int inner, group, room, groups, k_tiles, blocks;           // blocks of MX4_ROWS_THREADS a matrix
  int left_out;                  // matrices with so many slots or fewer are left out
  uint4* out;
};
__device__ __forceinline__ void mx4_gated_scales(const Mx4GatedScales& g, const int* __restrict__ plan, int matrix, int block) {
  if (plan[1 + matrix + 1] - plan[1 + matrix] <= g.left_out) return;
  const int tiles = g.groups * (g.room / 128), item = block * MX4_ROWS_THREADS + threadIdx.x;
  if (item >= tiles * g.k_tiles * 32) return;
  const int kt = item / 32 % g.k_tiles, tile = item / 32 / g.k_tiles;
  const size_t from = (size_t)matrix * mx4_tiles(2 * g.inner) * g.k_tiles * MX4_TILE_BYTES;
  unsigned w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = tile * 128 + q * 32 + (item & 31), n = row % g.room, feature = row / g.room * g.group + (n < g.group ? n : n - g.group);
    w[q] = n < 2 * g.group && feature < g.inner
               ? g.scales[(from + mx4_scale_word(n < g.group ? feature : g.inner + feature, kt, g.k_tiles)) / 4] : 0x7f7f7f7fu;
  }
  g.out[((size_t)(matrix * tiles + tile) * g.k_tiles + kt) * (MX4_TILE_BYTES / 16) + (item & 31)] = make_uint4(w[0], w[1], w[2], w[3]);
}
__global__ void __launch_bounds__(MX4_ROWS_THREADS) mx4_gated_scales_kernel(const Mx4GatedScales g, const int* __restrict__ plan) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  mx4_gated_scales(g, plan, blockIdx.x / g.blocks, blockIdx.x % g.blocks);
}

// The split into the order of a plan's tiles (csrc/moe.cu) of 256 slots, with room for 256 rows a tile: parts [2, 256 tiles, ...].  16 lanes have
// four column tiles of a row, their loads in flight together, split them once and store them for every choice of the row whose slot is in a tile (2,048
// rows of 2,048 with 6 choices: 16 us; slot by slot, each splitting again, 28).  The blocks behind those regroup scales (`g`; both are
// ahead of the same product, and one launch takes less than two).
#define MX4_SPLIT_AT_ONCE 4
template <bool WIDE>
__global__ void __launch_bounds__(MX4_ROWS_THREADS)
mx4_split_slots_kernel(const __nv_bfloat16* __restrict__ x, int rows, int width, const int* __restrict__ plan, const int* __restrict__ entry_slot, int top,
                       int experts, int max_tiles, int split_blocks, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales, const Mx4GatedScales g) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  if ((int)blockIdx.x >= split_blocks) {
    const int item = blockIdx.x - split_blocks;
    mx4_gated_scales(g, plan, item / g.blocks, item % g.blocks);
    return;
  }
  const int k_tiles = mx4_tiles(width), k_pieces = (k_tiles + MX4_SPLIT_AT_ONCE - 1) / MX4_SPLIT_AT_ONCE, lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_ROWS_THREADS / 16) + (threadIdx.x >> 4);
  const int kt0 = (int)(item % k_pieces) * MX4_SPLIT_AT_ONCE;
  const bool live = item / k_pieces < rows;
  const int row = live ? (int)(item / k_pieces) : rows - 1;
  const __nv_bfloat16* src = x + (size_t)row * width + kt0 * 128 + lane * 8;
  float v[MX4_SPLIT_AT_ONCE][8];
  if (WIDE && (kt0 + MX4_SPLIT_AT_ONCE) * 128 <= width) {
    uint4 raw[MX4_SPLIT_AT_ONCE];
#pragma unroll
    for (int j = 0; j < MX4_SPLIT_AT_ONCE; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + j * 128);
#pragma unroll
    for (int j = 0; j < MX4_SPLIT_AT_ONCE; ++j) mx4_unpack_bf16(raw[j], v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < MX4_SPLIT_AT_ONCE; ++j) mx4_load_eight<WIDE>(src + j * 128, width - (kt0 + j) * 128 - lane * 8, true, v[j]);
  }
  Mx4SplitEight e[MX4_SPLIT_AT_ONCE];
#pragma unroll
  for (int j = 0; j < MX4_SPLIT_AT_ONCE; ++j) e[j] = mx4_split_eight(v[j], lane);
  const int* tiles = plan + 1 + experts + 1;                 // (expert, first slot) of each, in the slots' order
  const size_t part = (size_t)max_tiles * 256 * k_tiles * 128, scale_part = (size_t)max_tiles * 2 * k_tiles * MX4_TILE_BYTES;
  for (int first = 0; first < top; first += 16) {
    // a choice a lane: the row of the tiles where it goes, if its slot is in one
    int to = -1;
    if (live && first + lane < top) {
      const int slot = entry_slot[(size_t)row * top + first + lane];
      int low = 0, high = slot < 0 ? 0 : plan[0];            // the first tile that begins behind the slot is among low .. high
      while (low < high) {
        const int middle = (low + high) / 2;
        if (tiles[2 * middle + 1] <= slot) low = middle + 1;
        else high = middle;
      }
      if (low > 0 && slot >= 0) {
        const int tile = low - 1, in_tile = slot - tiles[2 * tile + 1];
        if (in_tile < 256 && slot < plan[1 + tiles[2 * tile] + 1]) to = tile * 256 + in_tile;
      }
    }
    const int count = min(16, top - first);
    for (int i = 0; i < count; ++i) {
      const int dst = __shfl_sync(0xffffffffu, to, i, 16);
      if (dst < 0) continue;
#pragma unroll
      for (int j = 0; j < MX4_SPLIT_AT_ONCE; ++j)
        if (kt0 + j < k_tiles)
          mx4_store_split(e[j], lane, parts + ((size_t)dst * k_tiles + kt0 + j) * 128 + lane * 8, part, scales + mx4_scale_word(dst, kt0 + j, k_tiles), scale_part);
    }
  }
}

// Eight entries of 128 of a row (lane of 16) as the eight four-bit parts of mx4.cuh, rows of their own from `row` on.
template <bool WIDE>
__device__ __forceinline__ void mx4_parts_of_eight(const __nv_bfloat16* __restrict__ src, int left, bool live, int lane, int row, int kt, int k_tiles,
                                                   unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
  float v[8];
  mx4_load_eight<WIDE>(src, left, live, v);
  unsigned most = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned first = mx4_first_scale(most);
  // the first scales of the four blocks, a byte each, in one word: that of a later part is 3 less in each byte
  unsigned word = first << (8 * (lane >> 2));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = mx4_over_first_scale(v[i], first);
#pragma unroll
  for (int part = 0; part < MX4_PARTS; ++part) codes[((size_t)(row + part) * k_tiles + kt) * 16 + lane] = mx4_next_part(v);
  if (lane < MX4_PARTS) {
    unsigned mine = 0u;
#pragma unroll
    for (int b = 0; b < 4; ++b) mine |= mx4_part_scale((word >> (8 * b)) & 255u, lane) << (8 * b);
    *reinterpret_cast<unsigned*>(scales + mx4_scale_word(row + lane, kt, k_tiles)) = mine;
  }
}

// Rows of bfloat16 as parts: a matrix of 8 * rows rows in four bits, row 8 r + p the part p of row r.
template <bool WIDE>
__global__ void __launch_bounds__(MX4_ROWS_THREADS)
mx4_parts_kernel(const __nv_bfloat16* __restrict__ x, size_t pitch, int rows, int width, unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
  srb_grid_dependency_wait();
  srb_launch_dependents();                                  // (only now: the product starts on what is older than this kernel)
  const int k_tiles = mx4_tiles(width), lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_ROWS_THREADS / 16) + (threadIdx.x >> 4);
  const int row = (int)(item / k_tiles), kt = (int)(item % k_tiles), k = kt * 128 + lane * 8;
  mx4_parts_of_eight<WIDE>(x + (size_t)row * pitch + k, width - k, row < rows, lane, row * MX4_PARTS, kt, k_tiles, codes, scales);
}

// The same of the slots of a plan's tiles (of 8 slots): row (8 tile + place) * 8 + p.  A block has a tile's 128 entries.
template <bool WIDE>
__global__ void __launch_bounds__(128)
mx4_parts_slots_kernel(const __nv_bfloat16* __restrict__ x, int width, const int* __restrict__ plan, const int* __restrict__ slot_row, int experts,
                       unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
  srb_grid_dependency_wait();
  srb_launch_dependents();                                  // (only now: the product starts on what is older than this kernel)
  const int k_tiles = mx4_tiles(width), tile = blockIdx.x / k_tiles, kt = blockIdx.x % k_tiles, in_tile = threadIdx.x >> 4, lane = threadIdx.x & 15;
  if (tile >= plan[0]) return;
  const int expert = plan[1 + experts + 1 + 2 * tile], slot = plan[1 + experts + 1 + 2 * tile + 1] + in_tile;
  const bool live = slot < plan[1 + expert + 1];
  const int k = kt * 128 + lane * 8;
  mx4_parts_of_eight<WIDE>(x + (size_t)(live ? slot_row[slot] : 0) * width + k, width - k, live, lane, (tile * 8 + in_tile) * MX4_PARTS, kt, k_tiles,
                           codes, scales);
}

// out[row, :] = sum over the row's choices, in their order, of weight * y[slot, :], in 32 bits, rounded once.  Bound by the bytes of y: four
// columns a thread, the loads of eight choices in flight.
#define MX4_COMBINE_AT_ONCE 8
template <bool WIDE>
__global__ void __launch_bounds__(128)
mx4_combine_kernel(const float* __restrict__ y, const int* __restrict__ entry_slot, const float* __restrict__ weights, int top, int width,
                   __nv_bfloat16* __restrict__ out) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int row = blockIdx.x, i = (blockIdx.y * 128 + threadIdx.x) * 4;
  if (i >= width) return;
  const int* slots = entry_slot + (size_t)row * top;
  const float* w = weights + (size_t)row * top;
  float sum[4] = {};
  for (int first = 0; first < top; first += MX4_COMBINE_AT_ONCE) {
    float v[MX4_COMBINE_AT_ONCE][4], by[MX4_COMBINE_AT_ONCE];
#pragma unroll
    for (int k = 0; k < MX4_COMBINE_AT_ONCE; ++k) {
      const int slot = first + k < top ? slots[first + k] : -1;
      by[k] = slot >= 0 ? w[first + k] : 0.f;
      const float* src = y + (size_t)max(slot, 0) * width + i;
      if (slot < 0) {
        v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.f;
      } else if (WIDE) {
        const float4 q = *reinterpret_cast<const float4*>(src);
        v[k][0] = q.x; v[k][1] = q.y; v[k][2] = q.z; v[k][3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = i + j < width ? src[j] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < MX4_COMBINE_AT_ONCE; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = fmaf(by[k], v[k][j], sum[j]);
  }
  __nv_bfloat16* dst = out + (size_t)row * width + i;
  if (WIDE) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(sum[0], sum[1]), b = __floats2bfloat162_rn(sum[2], sum[3]);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < width) dst[j] = __float2bfloat16_rn(sum[j]);
  }
}
// ---- launches --------------------------------------------------------------------------------------------------------
static inline bool mx4_wide(const void* x, long long pitch) { return ((uintptr_t)x & 15) == 0 && pitch % 8 == 0; }
// 16 lanes for 128 entries of a row
static int mx4_rows_grid(long long rows, int width, dim3* grid) {
  const long long blocks = (rows * mx4_tiles(width) + MX4_ROWS_THREADS / 16 - 1) / (MX4_ROWS_THREADS / 16);
  if (blocks > 0x7fffffffll) SRB_FAIL("four-bit products: %lld rows of %d entries are too many", rows, width);
  *grid = dim3((unsigned)blocks);
  return SRB_OK;
}

// Two eight-bit parts: parts [2, rows, 128 column tiles], scales [2, row tiles, column tiles, 512].
static inline int mx4_launch_split(const void* x, long long pitch, int rows, int width, uint8_t* parts, uint8_t* scales, cudaStream_t s) {
  dim3 grid;
  if (mx4_rows_grid(rows, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  SRB_CUDA_CALL(srb_launch(mx4_wide(x, pitch) ? mx4_split_kernel<true> : mx4_split_kernel<false>, grid, dim3(MX4_ROWS_THREADS), 0, s,
                           (const __nv_bfloat16*)x, (size_t)pitch, rows, width, parts, scales));
  return SRB_OK;
}
// Eight four-bit parts: codes [8 rows, 64 column tiles] and the tiles of scales of 8 rows rows.
static inline int mx4_launch_parts(const void* x, long long pitch, int rows, int width, uint8_t* codes, uint8_t* scales, cudaStream_t s) {
  dim3 grid;
  if (mx4_rows_grid(rows, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  SRB_CUDA_CALL(srb_launch(mx4_wide(x, pitch) ? mx4_parts_kernel<true> : mx4_parts_kernel<false>, grid, dim3(MX4_ROWS_THREADS), 0, s,
                           (const __nv_bfloat16*)x, (size_t)pitch, rows, width, (unsigned*)codes, scales));
  return SRB_OK;
}
static inline int mx4_launch_parts_slots(const void* x, int width, const int* plan, const int* slot_row, int experts, int max_tiles, uint8_t* codes,
                                  uint8_t* scales, cudaStream_t s) {
  const long long blocks = (long long)max_tiles * mx4_tiles(width);
  if (max_tiles > 1 << 24 || blocks > 0x7fffffff) SRB_FAIL("four-bit experts: %d tiles are too many", max_tiles);
  SRB_CUDA_CALL(srb_launch(mx4_wide(x, width) ? mx4_parts_slots_kernel<true> : mx4_parts_slots_kernel<false>, dim3((unsigned)blocks),
                           dim3(128), 0, s, (const __nv_bfloat16*)x, width, plan, slot_row, experts, (unsigned*)codes, scales));
  return SRB_OK;
}
static inline size_t mx4_gated_scales_bytes(int matrices, int width, int room, int groups) {
  return (size_t)matrices * groups * (room / 128) * mx4_tiles(width) * MX4_TILE_BYTES;
}
static inline int mx4_make_gated_scales(Mx4GatedScales* g, const void* scales, int matrices, int inner, int width, int group, int room, int groups,
                                        int left_out, uint8_t* out) {
  const long long items = (long long)groups * (room / 128) * mx4_tiles(width) * 32, blocks = (items + MX4_ROWS_THREADS - 1) / MX4_ROWS_THREADS;
  if (items > 0x3fffffff || blocks * matrices > 0x3fffffff) SRB_FAIL("four-bit experts: %d matrices of 2 x %d rows of %d are too many", matrices, inner, width);
  *g = {(const unsigned*)scales, inner, group, room, groups, mx4_tiles(width), (int)blocks, left_out, (uint4*)out};
  return SRB_OK;
}
static inline int mx4_launch_gated_scales(const Mx4GatedScales& g, int matrices, const int* plan, cudaStream_t s) {
  SRB_CUDA_CALL(srb_launch(mx4_gated_scales_kernel, dim3(g.blocks * matrices), dim3(MX4_ROWS_THREADS), 0, s, g, plan));
  return SRB_OK;
}
// `g`: scales to be regrouped beside it, of `matrices` matrices (none: 0).
static inline int mx4_launch_split_slots(const void* x, int rows, int width, const int* plan, const int* entry_slot, int top, int experts, int max_tiles,
                                         uint8_t* parts, uint8_t* scales, const Mx4GatedScales& g, int matrices, cudaStream_t s) {
  const long long pieces = (mx4_tiles(width) + MX4_SPLIT_AT_ONCE - 1) / MX4_SPLIT_AT_ONCE;
  const long long blocks = (rows * pieces + MX4_ROWS_THREADS / 16 - 1) / (MX4_ROWS_THREADS / 16);
  if (max_tiles > 1 << 22 || blocks > 0x3fffffff) SRB_FAIL("four-bit experts: %d rows of %d, %d tiles are too many", rows, width, max_tiles);
  SRB_CUDA_CALL(srb_launch(mx4_wide(x, width) ? mx4_split_slots_kernel<true> : mx4_split_slots_kernel<false>, dim3((unsigned)(blocks + g.blocks * matrices)),
                           dim3(MX4_ROWS_THREADS), 0, s, (const __nv_bfloat16*)x, rows, width, plan, entry_slot, top, experts, max_tiles, (int)blocks, parts,
                           scales, g));
  return SRB_OK;
}
static inline int mx4_launch_combine(const float* y, const int* entry_slot, const float* weights, int rows, int top, int width, void* out, cudaStream_t s) {
  const bool wide = width % 4 == 0 && (((uintptr_t)y & 15) | ((uintptr_t)out & 7)) == 0;
  const int pieces = (width + 511) / 512;
  if (pieces > 65535) SRB_FAIL("four-bit experts: rows of %d are too wide", width);
  SRB_CUDA_CALL(srb_launch(wide ? mx4_combine_kernel<true> : mx4_combine_kernel<false>, dim3(rows, pieces), dim3(128), 0, s, y, entry_slot, weights,
                           top, width, (__nv_bfloat16*)out));
  return SRB_OK;
}

// Pieces of a caller's scratch memory, on 256-byte borders.
struct Mx4Scratch {
  uint8_t* base;
  size_t used;
  uint8_t* take(size_t bytes) {
    uint8_t* at = base + used;
    used += (bytes + 255) & ~(size_t)255;
    return at;
  }
};

// What a call on the experts has, for both libraries.
struct Mx4ExpertsCall {
  const void* h;                 // bfloat16 rows of `width`
  const int* plan;
  const void *up, *up_scales;    // [experts, 2 * inner or inner, width]
  const void *down, *down_scales;// [experts, width, inner]
  float* y;                      // [slots, width]
  int max_tiles, slots, experts, width, inner, gated, activation;
  float act_param;
  int* error_word;
  cudaStream_t stream;
};
static inline int mx4_check_experts(const Mx4ExpertsCall& c) {
  if (c.width <= 0 || c.inner <= 0) SRB_FAIL("four-bit experts: sizes %d, %d must be positive", c.width, c.inner);
  if (c.activation < 0 || c.activation >= SRB_ACT_COUNT) SRB_FAIL("four-bit experts: unknown activation %d", c.activation);
  if (((uintptr_t)c.up | (uintptr_t)c.down) & 31) SRB_FAIL("four-bit experts: codes must start on 32-byte borders");
  return SRB_OK;
}
