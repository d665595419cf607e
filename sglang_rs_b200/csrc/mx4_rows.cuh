// Around the products with four-bit matrices: rows of bfloat16 as the parts that multiply four-bit entries, the scales of stacked gate and up rows
// regrouped, and the weighted sum of the experts' results.  Kernels and their launches, for the two libraries that have products.
#pragma once
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"

#define MX4_ROWS_THREADS 256

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

// Eight entries of 128 of a row (lane of 16) as the two eight-bit parts of mx4.cuh, to `dst` and `dst + part`, and the row's scale words.
template <bool WIDE>
__device__ __forceinline__ void mx4_split_eight(const __nv_bfloat16* __restrict__ src, int left, bool live, int lane, uint8_t* dst, size_t part,
                                                uint8_t* word, size_t scale_part) {
  float v[8];
  mx4_load_eight<WIDE>(src, left, live, v);
  unsigned most = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned high = mx8_scale_high(most), low = mx8_scale_low(high);
  unsigned h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mx8_split(v[2 * i], v[2 * i + 1], high, low, h[i], l[i]);
  unsigned high_word = (lane & 3) == 0 ? high << (8 * (lane >> 2)) : 0u, low_word = (lane & 3) == 0 ? low << (8 * (lane >> 2)) : 0u;
#pragma unroll
  for (int offset = 4; offset <= 8; offset <<= 1) {
    high_word |= __shfl_xor_sync(0xffffffffu, high_word, offset);
    low_word |= __shfl_xor_sync(0xffffffffu, low_word, offset);
  }
  if (!live) return;
  *reinterpret_cast<uint2*>(dst) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  *reinterpret_cast<uint2*>(dst + part) = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
  if (lane == 0) {
    *reinterpret_cast<unsigned*>(word) = high_word;
    *reinterpret_cast<unsigned*>(word + scale_part) = low_word;
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
  mx4_split_eight<WIDE>(x + (size_t)row * pitch + k, width - k, row < rows, lane, parts + ((size_t)row * k_tiles * 128 + k),
                        (size_t)rows * k_tiles * 128, scales + mx4_scale_word(row, kt, k_tiles),
                        (size_t)mx4_tiles(rows) * k_tiles * MX4_TILE_BYTES);
}

// The same in the order of a plan's tiles (csrc/moe.cu) of 256 slots, with room for 256 rows a tile: parts [2, 256 tiles, ...].  16 lanes a
// slot, 16 slots a block.
template <bool WIDE>
__global__ void __launch_bounds__(MX4_ROWS_THREADS)
mx4_split_slots_kernel(const __nv_bfloat16* __restrict__ x, int width, const int* __restrict__ plan, const int* __restrict__ slot_row, int experts,
                       int max_tiles, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int tile = blockIdx.x / 16, in_tile = blockIdx.x % 16 * (MX4_ROWS_THREADS / 16) + (threadIdx.x >> 4), lane = threadIdx.x & 15;
  if (tile >= plan[0]) return;
  const int expert = plan[1 + experts + 1 + 2 * tile], slot = plan[1 + experts + 1 + 2 * tile + 1] + in_tile;
  const int end = plan[1 + expert + 1];                      // (a tile's place is below 256)
  if (slot - (in_tile & 1) >= end) return;                   // neither half of the warp has a slot
  const bool live = slot < end;
  const int k_tiles = mx4_tiles(width), row = tile * 256 + in_tile;
  const size_t part = (size_t)max_tiles * 256 * k_tiles * 128, scale_part = (size_t)max_tiles * 2 * k_tiles * MX4_TILE_BYTES;
  const __nv_bfloat16* src = x + (size_t)(live ? slot_row[slot] : 0) * width + lane * 8;
  uint8_t* dst = parts + ((size_t)row * k_tiles * 128 + lane * 8);
#pragma unroll 4
  for (int kt = 0; kt < k_tiles; ++kt)
    mx4_split_eight<WIDE>(src + kt * 128, width - kt * 128 - lane * 8, live, lane, dst + kt * 128, part, scales + mx4_scale_word(row, kt, k_tiles),
                          scale_part);
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

// Scales of stacked gate and up rows (2 * inner rows a matrix) in groups: `group` gate rows, the `group` up rows of the same features, room for
// `room` rows (a multiple of 128) a group.  A product tile's scales are whole tiles then, wherever the up rows begin.  Matrices without a slot in
// the plan are left out.  A thread has the 16 bytes of four rows, 32 apart.
__global__ void __launch_bounds__(MX4_ROWS_THREADS)
mx4_gated_scales_kernel(const unsigned* __restrict__ scales, int inner, int group, int room, int groups, int k_tiles, const int* __restrict__ plan,
                        uint4* __restrict__ out) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int matrix = blockIdx.y;
  if (plan[1 + matrix] == plan[1 + matrix + 1]) return;
  const int tiles = groups * (room / 128), item = blockIdx.x * MX4_ROWS_THREADS + threadIdx.x;
  if (item >= tiles * k_tiles * 32) return;
  const int kt = item / 32 % k_tiles, tile = item / 32 / k_tiles;
  const size_t from = (size_t)matrix * mx4_tiles(2 * inner) * k_tiles * MX4_TILE_BYTES;
  unsigned w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = tile * 128 + q * 32 + (item & 31), n = row % room, feature = row / room * group + (n < group ? n : n - group);
    w[q] = n < 2 * group && feature < inner ? scales[(from + mx4_scale_word(n < group ? feature : inner + feature, kt, k_tiles)) / 4] : 0x7f7f7f7fu;
  }
  out[((size_t)(matrix * tiles + tile) * k_tiles + kt) * (MX4_TILE_BYTES / 16) + (item & 31)] = make_uint4(w[0], w[1], w[2], w[3]);
}

// out[row, :] = sum over the row's choices, in their order, of weight * y[slot, :], in 32 bits, rounded once.  Bound by the bytes of y: four
// columns a thread, the loads of four choices in flight.
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
  for (int first = 0; first < top; first += 4) {
    float v[4][4], by[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
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
    for (int k = 0; k < 4; ++k)
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
static inline int mx4_launch_split_slots(const void* x, int width, const int* plan, const int* slot_row, int experts, int max_tiles, uint8_t* parts,
                                  uint8_t* scales, cudaStream_t s) {
  if (max_tiles > 1 << 22) SRB_FAIL("four-bit experts: %d tiles are too many", max_tiles);
  SRB_CUDA_CALL(srb_launch(mx4_wide(x, width) ? mx4_split_slots_kernel<true> : mx4_split_slots_kernel<false>, dim3(256 / 16 * max_tiles),
                           dim3(MX4_ROWS_THREADS), 0, s, (const __nv_bfloat16*)x, width, plan, slot_row, experts, max_tiles, parts, scales));
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
static inline int mx4_launch_gated_scales(const void* scales, int matrices, int inner, int width, int group, int room, int groups, const int* plan,
                                   uint8_t* out, cudaStream_t s) {
  const long long items = (long long)groups * (room / 128) * mx4_tiles(width) * 32;
  if (matrices > 65535 || items > 0x3fffffff) SRB_FAIL("four-bit experts: %d matrices of 2 x %d rows of %d are too many", matrices, inner, width);
  SRB_CUDA_CALL(srb_launch(mx4_gated_scales_kernel, dim3((unsigned)((items + MX4_ROWS_THREADS - 1) / MX4_ROWS_THREADS), matrices),
                           dim3(MX4_ROWS_THREADS), 0, s, (const unsigned*)scales, inner, group, room, groups, mx4_tiles(width), plan, (uint4*)out));
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
  const int *plan, *slot_row;
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
