// Rows into the microscaled four-bit format of mx4.cuh and back.
//
//   srb_mx4_quantize     per block of 32 entries: e = floor(log2(largest magnitude)) - 2, at least -127; s = e + 127; an entry is
//                        x / 2^e rounded to the nearest value, ties to the even mantissa, magnitudes above 6 to 6 (the OCP
//                        specification's conversion).  x / 2^e is exact, so the codes are a function of the numbers alone.  A block
//                        that holds an infinity or something that is not a number has s = 255 and codes of zero.
//   srb_mx4_dequantize   the values, in bfloat16 (which holds every one of them exactly) or float.
//
// Both are bound by the bytes of the wide side.  A row's 128 entries are the work of 16 lanes, 8 entries (16 bytes of bfloat16) each; 4 lanes
// are a block.
#include "common.cuh"
#include "mx4.cuh"

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MX4_THREADS 256

__device__ __forceinline__ void mx4_unpack_bf16(const uint4& raw, float (&v)[8]) {
  const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_quantize_kernel(const T* __restrict__ x, size_t pitch, size_t matrix_pitch, int rows, int width, unsigned* __restrict__ codes,
                    unsigned* __restrict__ scales) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), row_tiles = mx4_tiles(rows);
  const int lane = threadIdx.x & 15;                         // of the 16 that share 128 entries of a row
  const long long item = (long long)blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4);
  const int row = (int)(item / k_tiles), kt = (int)(item % k_tiles), matrix = blockIdx.y;
  const bool inside = row < row_tiles * 128, live = row < rows;
  const int k = kt * 128 + lane * 8;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (live) {
    const T* src = x + (size_t)matrix * matrix_pitch + (size_t)row * pitch + k;
    if (WIDE && k + 8 <= width) {
      if (sizeof(T) == 2) mx4_unpack_bf16(*reinterpret_cast<const uint4*>(src), v);
      else {
        const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < width) v[i] = srb_to_float(src[i]);
    }
  }
  // magnitudes as their bits: the largest bits are the largest magnitude, and whatever is not finite is above all that is
  unsigned most = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const bool finite = most < 0x7f800000u;
  const int exponent = max((int)(most >> 23) - 129, -127);   // a subnormal's field is 0: the least scale
  const unsigned s = finite ? (unsigned)(exponent + 127) : 255u;
  const float inverse = __uint_as_float((unsigned)(127 - exponent) << 23);      // 2^-exponent, between 2^-125 and 2^127
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = finite ? v[i] * inverse : 0.f;
  const unsigned packed = mx4_pack_eight(v);
  // the scales of the four blocks, a byte each, in one word; blocks behind the row's end and rows behind the last get 127
  unsigned word = live && kt * 128 + (lane >> 2) * 32 < width ? s : 127u;
  word = (lane & 3) == 0 ? word << (8 * (lane >> 2)) : 0u;
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (!inside) return;
  if (live) codes[((size_t)matrix * rows + row) * (mx4_pitch(width) / 4) + kt * 16 + lane] = packed;
  if (lane == 0) scales[((size_t)matrix * row_tiles * k_tiles * MX4_TILE_BYTES + mx4_scale_word(row, kt, k_tiles)) / 4] = word;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_dequantize_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ scales, int rows, int width, T* __restrict__ out) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), row_tiles = mx4_tiles(rows);
  const int lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4);
  const int row = (int)(item / k_tiles), kt = (int)(item % k_tiles), matrix = blockIdx.y;
  if (row >= rows) return;
  const unsigned packed = codes[((size_t)matrix * rows + row) * (mx4_pitch(width) / 4) + kt * 16 + lane];
  const unsigned word = scales[((size_t)matrix * row_tiles * k_tiles * MX4_TILE_BYTES + mx4_scale_word(row, kt, k_tiles)) / 4];
  const float scale = mx4_scale_value((word >> (8 * (lane >> 2))) & 255u);
  const int k = kt * 128 + lane * 8;
  T* dst = out + ((size_t)matrix * rows + row) * width + k;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = mx4_code_value((packed >> (4 * i)) & 15u) * scale;
  if (WIDE && k + 8 <= width) {
    if (sizeof(T) == 2) {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&pair);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < width) dst[i] = srb_from_float<T>(v[i]);
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
__global__ void __launch_bounds__(MX4_THREADS)
mx4_split_kernel(const __nv_bfloat16* __restrict__ x, size_t pitch, int rows, int width, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4);
  const int row = (int)(item / k_tiles), kt = (int)(item % k_tiles), k = kt * 128 + lane * 8;
  mx4_split_eight<WIDE>(x + (size_t)row * pitch + k, width - k, row < rows, lane, parts + ((size_t)row * k_tiles * 128 + k),
                        (size_t)rows * k_tiles * 128, scales + mx4_scale_word(row, kt, k_tiles),
                        (size_t)mx4_tiles(rows) * k_tiles * MX4_TILE_BYTES);
}

// The same in the order of a plan's tiles (csrc/moe.cu) of 256 slots, with room for 256 rows a tile: parts [2, 256 tiles, ...].  16 lanes a
// slot, 16 slots a block.
template <bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_split_slots_kernel(const __nv_bfloat16* __restrict__ x, int width, const int* __restrict__ plan, const int* __restrict__ slot_row, int experts,
                       int max_tiles, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int tile = blockIdx.y, in_tile = blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4), lane = threadIdx.x & 15;
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
__global__ void __launch_bounds__(MX4_THREADS)
mx4_parts_kernel(const __nv_bfloat16* __restrict__ x, size_t pitch, int rows, int width, unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
  srb_grid_dependency_wait();
  srb_launch_dependents();                                  // (only now: the product starts on what is older than this kernel)
  const int k_tiles = mx4_tiles(width), lane = threadIdx.x & 15;
  const long long item = (long long)blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4);
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
  const int tile = blockIdx.y, kt = blockIdx.x, in_tile = threadIdx.x >> 4, lane = threadIdx.x & 15;
  if (tile >= plan[0]) return;
  const int expert = plan[1 + experts + 1 + 2 * tile], slot = plan[1 + experts + 1 + 2 * tile + 1] + in_tile;
  const bool live = slot < plan[1 + expert + 1];
  const int k = kt * 128 + lane * 8;
  mx4_parts_of_eight<WIDE>(x + (size_t)(live ? slot_row[slot] : 0) * width + k, width - k, live, lane, (tile * 8 + in_tile) * MX4_PARTS, kt, gridDim.x,
                           codes, scales);
}

// Scales of stacked gate and up rows (2 * inner rows a matrix) in groups: `group` gate rows, the `group` up rows of the same features, room for
// `room` rows (a multiple of 128) a group.  A product tile's scales are whole tiles then, wherever the up rows begin.  Matrices without a slot in
// the plan are left out.  A thread has the 16 bytes of four rows, 32 apart.
__global__ void __launch_bounds__(MX4_THREADS)
mx4_gated_scales_kernel(const unsigned* __restrict__ scales, int inner, int group, int room, int groups, int k_tiles, const int* __restrict__ plan,
                        uint4* __restrict__ out) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int matrix = blockIdx.y;
  if (plan[1 + matrix] == plan[1 + matrix + 1]) return;
  const int tiles = groups * (room / 128), item = blockIdx.x * MX4_THREADS + threadIdx.x;
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

static int mx4_grid(int matrices, long long rows, int width, dim3* grid) {
  const long long items = rows * mx4_tiles(width), blocks = (items + MX4_THREADS / 16 - 1) / (MX4_THREADS / 16);
  if (blocks > 0x7fffffffll || matrices > 65535) SRB_FAIL("mx4: %d matrices of %lld rows of %d entries are too many", matrices, rows, width);
  *grid = dim3((unsigned)blocks, (unsigned)matrices);
  return SRB_OK;
}

// x: `matrices` matrices, `matrix_pitch` elements apart, of `rows` rows, `pitch` elements apart, of `width` entries.
extern "C" int srb_mx4_quantize(const void* x, long long pitch, long long matrix_pitch, int matrices, int rows, int width, void* codes,
                                void* scales, int dtype, void* stream) {
  if (matrices <= 0 || rows <= 0 || width <= 0) return SRB_OK;
  dim3 grid;
  if (mx4_grid(matrices, (long long)mx4_tiles(rows) * 128, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  const int element = dtype == SRB_DTYPE_F32 ? 4 : 2;
  const bool wide = ((uintptr_t)x & 15) == 0 && pitch * element % 16 == 0 && matrix_pitch * element % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SRB_DTYPE_F32)
    SRB_CUDA_CALL(srb_launch(wide ? mx4_quantize_kernel<float, true> : mx4_quantize_kernel<float, false>, grid, dim3(MX4_THREADS), 0, s,
                             (const float*)x, (size_t)pitch, (size_t)matrix_pitch, rows, width, (unsigned*)codes, (unsigned*)scales));
  else if (dtype == SRB_DTYPE_BF16)
    SRB_CUDA_CALL(srb_launch(wide ? mx4_quantize_kernel<__nv_bfloat16, true> : mx4_quantize_kernel<__nv_bfloat16, false>, grid, dim3(MX4_THREADS), 0,
                             s, (const __nv_bfloat16*)x, (size_t)pitch, (size_t)matrix_pitch, rows, width, (unsigned*)codes, (unsigned*)scales));
  else
    SRB_FAIL("mx4_quantize: unknown dtype %d", dtype);
  SRB_LAUNCH_CHECK("mx4_quantize");
  return SRB_OK;
}

extern "C" int srb_mx4_dequantize(const void* codes, const void* scales, int matrices, int rows, int width, void* out, int dtype, void* stream) {
  if (matrices <= 0 || rows <= 0 || width <= 0) return SRB_OK;
  dim3 grid;
  if (mx4_grid(matrices, rows, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  const int element = dtype == SRB_DTYPE_F32 ? 4 : 2;
  const bool wide = ((uintptr_t)out & 15) == 0 && (long long)width * element % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SRB_DTYPE_F32)
    SRB_CUDA_CALL(srb_launch(wide ? mx4_dequantize_kernel<float, true> : mx4_dequantize_kernel<float, false>, grid, dim3(MX4_THREADS), 0, s,
                             (const unsigned*)codes, (const unsigned*)scales, rows, width, (float*)out));
  else if (dtype == SRB_DTYPE_BF16)
    SRB_CUDA_CALL(srb_launch(wide ? mx4_dequantize_kernel<__nv_bfloat16, true> : mx4_dequantize_kernel<__nv_bfloat16, false>, grid,
                             dim3(MX4_THREADS), 0, s, (const unsigned*)codes, (const unsigned*)scales, rows, width, (__nv_bfloat16*)out));
  else
    SRB_FAIL("mx4_dequantize: unknown dtype %d", dtype);
  SRB_LAUNCH_CHECK("mx4_dequantize");
  return SRB_OK;
}

extern "C" int srb_mx4_split(const void* x, long long pitch, int rows, int width, void* parts, void* scales, void* stream) {
  if (rows <= 0 || width <= 0) return SRB_OK;
  dim3 grid;
  if (mx4_grid(1, rows, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  const bool wide = ((uintptr_t)x & 15) == 0 && pitch % 8 == 0;
  SRB_CUDA_CALL(srb_launch(wide ? mx4_split_kernel<true> : mx4_split_kernel<false>, grid, dim3(MX4_THREADS), 0, (cudaStream_t)stream,
                           (const __nv_bfloat16*)x, (size_t)pitch, rows, width, (uint8_t*)parts, (uint8_t*)scales));
  SRB_LAUNCH_CHECK("mx4_split");
  return SRB_OK;
}

extern "C" int srb_mx4_split_slots(const void* x, int width, const int* plan, const int* slot_row, int experts, int max_tiles,
                                   void* parts, void* scales, void* stream) {
  if (max_tiles <= 0 || width <= 0) return SRB_OK;
  if (max_tiles > 65535) SRB_FAIL("mx4_split_slots: %d tiles are too many", max_tiles);
  const bool wide = ((uintptr_t)x & 15) == 0 && width % 8 == 0;
  SRB_CUDA_CALL(srb_launch(wide ? mx4_split_slots_kernel<true> : mx4_split_slots_kernel<false>, dim3(256 / 16, max_tiles),
                           dim3(MX4_THREADS), 0, (cudaStream_t)stream, (const __nv_bfloat16*)x, width, plan, slot_row, experts, max_tiles,
                           (uint8_t*)parts, (uint8_t*)scales));
  SRB_LAUNCH_CHECK("mx4_split_slots");
  return SRB_OK;
}

extern "C" int srb_mx4_gated_scales(const void* scales, int matrices, int inner, int width, int group, int room, int groups, const int* plan,
                                    void* out, void* stream) {
  if (matrices <= 0 || inner <= 0 || width <= 0) return SRB_OK;
  const long long items = (long long)groups * (room / 128) * mx4_tiles(width) * 32;
  if (group <= 0 || room % 128 || room < 2 * group || matrices > 65535 || items > 0x3fffffff)
    SRB_FAIL("mx4_gated_scales: %d matrices, groups of %d in the room of %d", matrices, group, room);
  SRB_CUDA_CALL(srb_launch(mx4_gated_scales_kernel, dim3((unsigned)((items + MX4_THREADS - 1) / MX4_THREADS), matrices), dim3(MX4_THREADS), 0,
                           (cudaStream_t)stream, (const unsigned*)scales, inner, group, room, groups, mx4_tiles(width), plan, (uint4*)out));
  SRB_LAUNCH_CHECK("mx4_gated_scales");
  return SRB_OK;
}

// x [rows, width], `pitch` elements apart; codes [8 rows, 64 column tiles] and the tiles of scales of 8 rows rows.
extern "C" int srb_mx4_parts(const void* x, long long pitch, int rows, int width, void* codes, void* scales, void* stream) {
  if (rows <= 0 || width <= 0) return SRB_OK;
  dim3 grid;
  if (rows > 0x0fffffff || mx4_grid(1, rows, width, &grid) != SRB_OK) return SRB_ERR_INVALID;
  const bool wide = ((uintptr_t)x & 15) == 0 && pitch % 8 == 0;
  SRB_CUDA_CALL(srb_launch(wide ? mx4_parts_kernel<true> : mx4_parts_kernel<false>, grid, dim3(MX4_THREADS), 0, (cudaStream_t)stream,
                           (const __nv_bfloat16*)x, (size_t)pitch, rows, width, (unsigned*)codes, (uint8_t*)scales));
  SRB_LAUNCH_CHECK("mx4_parts");
  return SRB_OK;
}

// By the slots of a plan with tiles of 8 slots: codes [64 max_tiles, 64 column tiles].
extern "C" int srb_mx4_parts_slots(const void* x, int width, const int* plan, const int* slot_row, int experts, int max_tiles, void* codes,
                                   void* scales, void* stream) {
  if (max_tiles <= 0 || width <= 0) return SRB_OK;
  if (max_tiles > 65535) SRB_FAIL("mx4_parts_slots: %d tiles are too many", max_tiles);
  const bool wide = ((uintptr_t)x & 15) == 0 && width % 8 == 0;
  SRB_CUDA_CALL(srb_launch(wide ? mx4_parts_slots_kernel<true> : mx4_parts_slots_kernel<false>, dim3(mx4_tiles(width), max_tiles), dim3(128), 0,
                           (cudaStream_t)stream, (const __nv_bfloat16*)x, width, plan, slot_row, experts, (unsigned*)codes, (uint8_t*)scales));
  SRB_LAUNCH_CHECK("mx4_parts_slots");
  return SRB_OK;
}
