// Rows into the microscaled four-bit format of mx4.cuh and back.
//
//   srb_mx4_quantize     per block of 32 entries: e = floor(log2(largest magnitude)) - 2, at least -127; s = e + 127; an entry is
//                        x / 2^e rounded to the nearest value, ties to the even mantissa, magnitudes above 6 to 6 (the OCP
//                        specification's conversion).  x / 2^e is exact, so the codes are a function of the numbers alone.  A block
//                        that holds an infinity or something that is not a number has s = 255 and codes of zero.
//   srb_mx4_dequantize   the values, in bfloat16 or float, which hold all below 2^128 exactly.
//
// Both are bound by the bytes of the wide side: 2,048 rows of 12,288 bfloat16 there and back in 24 us, 0.80 of the measured copy rate (128 MB).  A
// row's 128 entries are the work of 16 lanes, 8 entries (16 bytes of bfloat16) each; 4 lanes are a block.
#include "common.cuh"
#include "mx4.cuh"

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MX4_THREADS 256

// Eight entries a lane, lane of 16, of a row's last 128 or of a row that does not start on a 16-byte border: through shared memory, so that neighbouring
// lanes read neighbouring entries (5,171 rows of 2,891 floats quantised and back: 34 us instead of 72).
template <typename T>
__device__ __forceinline__ void mx4_read_strided(const T* __restrict__ src, int left, int lane, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = lane + 16 * i < left ? srb_to_float(src[lane + 16 * i]) : 0.f;
}
__device__ __forceinline__ void mx4_turn(float* staged, int lane, float (&v)[8]) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) staged[lane + 16 * i] = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = staged[8 * lane + i];
}
__device__ __forceinline__ void mx4_unpack(const uint4 (&raw)[1], float (&v)[8]) { mx4_unpack_bf16(raw[0], v); }
__device__ __forceinline__ void mx4_unpack(const uint4 (&raw)[2], float (&v)[8]) {
  const unsigned w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}

// AT_ONCE column tiles of a row a thread takes: their loads are in flight together.
template <typename T, bool WIDE, int AT_ONCE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_quantize_kernel(const T* __restrict__ x, size_t pitch, size_t matrix_pitch, int rows, int width, unsigned* __restrict__ codes,
                    uint8_t* __restrict__ scales) {
  constexpr int PIECES = sizeof(T) / 2;                      // of 16 bytes, for eight entries
  __shared__ float staged[MX4_THREADS / 16][128 + 4];
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), row_tiles = mx4_tiles(rows);
  const int lane = threadIdx.x & 15, row = blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4), kt0 = blockIdx.y * AT_ONCE, matrix = blockIdx.z;
  const bool live = row < rows;
  const T* src = x + (size_t)matrix * matrix_pitch + (size_t)min(row, rows - 1) * pitch;
  auto store = [&](int kt, float (&v)[8]) {
    // magnitudes as their bits: the largest bits are the largest magnitude, and whatever is not finite is above all that is
    unsigned most = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const bool finite = most < 0x7f800000u;
    const unsigned s = finite ? max(most >> 23, 2u) - 2u : 255u;       // a subnormal's field is 0: the least scale
    const float inverse = __uint_as_float((254u - s) << 23); // 1 / 2^(s - 127), between 2^-125 and 2^127
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;
    const unsigned packed = finite ? mx4_pack_eight(v) : 0u;
    if (live) codes[((size_t)matrix * rows + row) * (mx4_pitch(width) / 4) + kt * 16 + lane] = packed;
    // a block's scale by its first lane; blocks behind the row's end and rows behind the last get 127
    if ((lane & 3) == 0)
      scales[(size_t)matrix * row_tiles * k_tiles * MX4_TILE_BYTES + mx4_scale_word(row, kt, k_tiles) + (lane >> 2)] =
          (uint8_t)(live && kt * 128 + lane * 8 < width ? s : 127u);
  };
  if (WIDE && (kt0 + AT_ONCE) * 128 <= width) {
    uint4 raw[AT_ONCE][PIECES];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) raw[j][i] = reinterpret_cast<const uint4*>(src + (kt0 + j) * 128)[PIECES * lane + i];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      float v[8];
      mx4_unpack(raw[j], v);
      store(kt0 + j, v);
    }
  } else {
    float v[AT_ONCE][8];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) mx4_read_strided(src + (kt0 + j) * 128, width - (kt0 + j) * 128, lane, v[j]);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (kt0 + j >= k_tiles) break;
      mx4_turn(staged[threadIdx.x >> 4], lane, v[j]);
      store(kt0 + j, v[j]);
    }
  }
}

template <typename T, bool WIDE, int AT_ONCE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_dequantize_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ scales, int rows, int width, T* __restrict__ out) {
  __shared__ float staged[MX4_THREADS / 16][128 + 4];
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int k_tiles = mx4_tiles(width), row_tiles = mx4_tiles(rows);
  const int lane = threadIdx.x & 15, row = blockIdx.x * (MX4_THREADS / 16) + (threadIdx.x >> 4), kt0 = blockIdx.y * AT_ONCE, matrix = blockIdx.z;
  const bool live = row < rows;
  unsigned packed[AT_ONCE], word[AT_ONCE];
#pragma unroll
  for (int j = 0; j < AT_ONCE; ++j) {
    const int kt = kt0 + j;
    packed[j] = live && kt < k_tiles ? codes[((size_t)matrix * rows + row) * (mx4_pitch(width) / 4) + kt * 16 + lane] : 0u;
    word[j] = live && kt < k_tiles ? scales[((size_t)matrix * row_tiles * k_tiles * MX4_TILE_BYTES + mx4_scale_word(row, kt, k_tiles)) / 4] : 0u;
  }
  T* dst = out + ((size_t)matrix * rows + row) * width;
#pragma unroll
  for (int j = 0; j < AT_ONCE; ++j) {
    const int k = (kt0 + j) * 128;
    if (k >= width) break;
    const float scale = mx4_scale_value((word[j] >> (8 * (lane >> 2))) & 255u);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) mx4_two_values((packed[j] >> (8 * i)) & 255u, v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
    if (WIDE && k + 128 <= width) {
      if (!live) continue;
      if (sizeof(T) == 2) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const unsigned*>(&pair);
        }
        reinterpret_cast<uint4*>(dst + k)[lane] = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        reinterpret_cast<float4*>(dst + k)[2 * lane] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst + k)[2 * lane + 1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
      float* mine = staged[threadIdx.x >> 4];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[8 * lane + i] = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (live && k + lane + 16 * i < width) dst[k + lane + 16 * i] = srb_from_float<T>(mine[lane + 16 * i]);
    }
  }
}

// Four tiles a thread where that leaves the SMs' threads busy, one otherwise (8 rows of 4,096: 1.8 us by one a thread, 2.9 by four; 2,048 rows of
// 12,288: 24.6 and 15.5).
static int mx4_grid(int matrices, int rows, int width, dim3* grid, int* at_once) {
  const long long k_tiles = mx4_tiles(width), row_blocks = (rows + MX4_THREADS / 16 - 1) / (MX4_THREADS / 16);
  *at_once = matrices * row_blocks * k_tiles >= 4ll * 8 * srb_sm_count() ? 4 : 1;
  const long long k_blocks = (k_tiles + *at_once - 1) / *at_once;
  if (k_blocks > 65535 || matrices > 65535) SRB_FAIL("mx4: %d matrices of %d rows of %d entries are too many", matrices, rows, width);
  *grid = dim3((unsigned)row_blocks, (unsigned)k_blocks, (unsigned)matrices);
  return SRB_OK;
}

template <typename T>
static int launch_quantize(const void* x, size_t pitch, size_t matrix_pitch, bool wide, int rows, int width, void* codes, void* scales, dim3 grid,
                           int at_once, cudaStream_t s) {
  auto kernel = wide ? (at_once == 4 ? mx4_quantize_kernel<T, true, 4> : mx4_quantize_kernel<T, true, 1>)
                     : (at_once == 4 ? mx4_quantize_kernel<T, false, 4> : mx4_quantize_kernel<T, false, 1>);
  SRB_CUDA_CALL(srb_launch(kernel, grid, dim3(MX4_THREADS), 0, s, (const T*)x, pitch, matrix_pitch, rows, width, (unsigned*)codes, (uint8_t*)scales));
  return SRB_OK;
}
template <typename T>
static int launch_dequantize(const void* codes, const void* scales, bool wide, int rows, int width, void* out, dim3 grid, int at_once, cudaStream_t s) {
  auto kernel = wide ? (at_once == 4 ? mx4_dequantize_kernel<T, true, 4> : mx4_dequantize_kernel<T, true, 1>)
                     : (at_once == 4 ? mx4_dequantize_kernel<T, false, 4> : mx4_dequantize_kernel<T, false, 1>);
  SRB_CUDA_CALL(srb_launch(kernel, grid, dim3(MX4_THREADS), 0, s, (const unsigned*)codes, (const unsigned*)scales, rows, width, (T*)out));
  return SRB_OK;
}

// x: `matrices` matrices, `matrix_pitch` elements apart, of `rows` rows, `pitch` elements apart, of `width` entries.
extern "C" int srb_mx4_quantize(const void* x, long long pitch, long long matrix_pitch, int matrices, int rows, int width, void* codes,
                                void* scales, int dtype, void* stream) {
  if (matrices <= 0 || rows <= 0 || width <= 0) return SRB_OK;
  if (dtype != SRB_DTYPE_F32 && dtype != SRB_DTYPE_BF16) SRB_FAIL("mx4_quantize: unknown dtype %d", dtype);
  if (rows > 0x7fff0000) SRB_FAIL("mx4_quantize: %d rows are too many", rows);
  dim3 grid;
  int at_once;
  if (mx4_grid(matrices, mx4_tiles(rows) * 128, width, &grid, &at_once) != SRB_OK) return SRB_ERR_INVALID;
  const int element = dtype == SRB_DTYPE_F32 ? 4 : 2;
  const bool wide = ((uintptr_t)x & 15) == 0 && pitch * element % 16 == 0 && matrix_pitch * element % 16 == 0;
  return dtype == SRB_DTYPE_F32
             ? launch_quantize<float>(x, (size_t)pitch, (size_t)matrix_pitch, wide, rows, width, codes, scales, grid, at_once, (cudaStream_t)stream)
             : launch_quantize<__nv_bfloat16>(x, (size_t)pitch, (size_t)matrix_pitch, wide, rows, width, codes, scales, grid, at_once, (cudaStream_t)stream);
}

extern "C" int srb_mx4_dequantize(const void* codes, const void* scales, int matrices, int rows, int width, void* out, int dtype, void* stream) {
  if (matrices <= 0 || rows <= 0 || width <= 0) return SRB_OK;
  if (dtype != SRB_DTYPE_F32 && dtype != SRB_DTYPE_BF16) SRB_FAIL("mx4_dequantize: unknown dtype %d", dtype);
  dim3 grid;
  int at_once;
  if (mx4_grid(matrices, rows, width, &grid, &at_once) != SRB_OK) return SRB_ERR_INVALID;
  const int element = dtype == SRB_DTYPE_F32 ? 4 : 2;
  const bool wide = ((uintptr_t)out & 15) == 0 && (long long)width * element % 16 == 0;
  return dtype == SRB_DTYPE_F32 ? launch_dequantize<float>(codes, scales, wide, rows, width, out, grid, at_once, (cudaStream_t)stream)
                                : launch_dequantize<__nv_bfloat16>(codes, scales, wide, rows, width, out, grid, at_once, (cudaStream_t)stream);
}
