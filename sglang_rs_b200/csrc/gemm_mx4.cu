// Y = X W^T with W in the microscaled four-bit format of mx4.cuh; X in bfloat16 or in that format too; sums in 32 bits.
//
// Tiles of 64 rows x 64 features by multiply-adds, both operands turned into floats on their way into shared memory.  Over experts
// (GROUPED) a tile is up to 64 slots of one expert, from the plan of csrc/moe.cu.
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MXG_TILE 64
#define MXG_BF16 0     // out bfloat16 = x w^T + bias
#define MXG_F32 1      // out float
#define MXG_GATED 2    // out bfloat16 = act(x gate^T) * (x up^T), the up rows `features` behind the gate rows
#define MXG_ACT 5      // out bfloat16 = act(x w^T)

struct Mx4Args {
  const void* x;               // bfloat16 rows, or codes
  const uint8_t* x_scales;     // of codes
  size_t ldx;                  // elements (bytes of codes) between rows
  const uint8_t* w;
  const uint8_t* w_scales;
  const float* bias;
  void* out;
  int rows, features, w_rows, width, activation;
  size_t ldo;
  float act_param;
  const int* plan;             // GROUPED
  const int* slot_row;         // rows of x are gathered by it, or are the slots themselves (null)
  int experts;
};

__device__ __forceinline__ float mxg_weight(const Mx4Args& a, int matrix, int row, int k) {
  if (row >= a.w_rows || k >= a.width) return 0.f;
  const int k_tiles = mx4_tiles(a.width);
  const unsigned byte = a.w[((size_t)matrix * a.w_rows + row) * mx4_pitch(a.width) + (k >> 1)];
  const unsigned s = a.w_scales[(size_t)matrix * mx4_tiles(a.w_rows) * k_tiles * MX4_TILE_BYTES + mx4_scale_word(row, k >> 7, k_tiles) + ((k >> 5) & 3)];
  return mx4_code_value(k & 1 ? byte >> 4 : byte & 15u) * mx4_scale_value(s);
}

template <bool FOUR, int MODE, bool GROUPED>
__global__ void __launch_bounds__(256) mx4_product_kernel(Mx4Args a) {
  __shared__ float xs[32][MXG_TILE + 4], ws[32][MXG_TILE + 4], us[MODE == MXG_GATED ? 32 : 1][MXG_TILE + 4];
  srb_launch_dependents();
  srb_grid_dependency_wait();
  int matrix = 0, first = blockIdx.y * MXG_TILE, count = min(MXG_TILE, a.rows - first);
  if (GROUPED) {
    if ((int)blockIdx.y >= a.plan[0]) return;
    const int* tiles = a.plan + 1 + a.experts + 1;
    matrix = tiles[2 * blockIdx.y];
    first = tiles[2 * blockIdx.y + 1];
    count = min(MXG_TILE, a.plan[1 + matrix + 1] - first);
  }
  const int feature0 = blockIdx.x * MXG_TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {}, acc_up[4][4] = {};
  for (int k0 = 0; k0 < a.width; k0 += 32) {
    for (int i = threadIdx.x; i < 32 * MXG_TILE; i += 256) {
      const int k = k0 + (i & 31), r = i >> 5;
      float v = 0.f;
      if (r < count && k < a.width) {
        const int row = GROUPED && a.slot_row ? a.slot_row[first + r] : first + r;
        if (FOUR) {
          const unsigned byte = reinterpret_cast<const uint8_t*>(a.x)[(size_t)row * a.ldx + (k >> 1)];
          const unsigned s = a.x_scales[mx4_scale_word(row, k >> 7, mx4_tiles(a.width)) + ((k >> 5) & 3)];
          v = mx4_code_value(k & 1 ? byte >> 4 : byte & 15u) * mx4_scale_value(s);
        } else {
          v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.x)[(size_t)row * a.ldx + k]);
        }
      }
      xs[i & 31][r] = v;
      ws[i & 31][r] = feature0 + r < a.features ? mxg_weight(a, matrix, feature0 + r, k) : 0.f;
      if (MODE == MXG_GATED) us[i & 31][r] = feature0 + r < a.features ? mxg_weight(a, matrix, a.features + feature0 + r, k) : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx * 4 + j], acc[i][j]);
          if (MODE == MXG_GATED) acc_up[i][j] = fmaf(xs[k][ty * 4 + i], us[k][tx * 4 + j], acc_up[i][j]);
        }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = ty * 4 + i, feature = feature0 + tx * 4 + j;
      if (r >= count || feature >= a.features) continue;
      float v = acc[i][j];
      if (MODE == MXG_GATED) v = srb_gated<true>(a.activation, v, acc_up[i][j], a.act_param);
      if (MODE == MXG_ACT) v = srb_gated<true>(a.activation, v, 1.0f, a.act_param);
      if (a.bias) v += a.bias[feature];
      const size_t at = (size_t)(first + r) * a.ldo + feature;
      if (MODE == MXG_F32) reinterpret_cast<float*>(a.out)[at] = v;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    }
}

// x [rows, width] bfloat16, `ldx` elements apart, or (x_scales given) codes; w_rows = features rows of codes and their scales; out [rows, ldo].
extern "C" int srb_mx4_linear(const void* x, const void* x_scales, long long ldx, const void* w, const void* w_scales, const float* bias,
                              void* out, long long ldo, int rows, int features, int width, int out_float, int* error_word, void* stream) {
  if (rows <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_linear: inner size %d must be positive", width);
  Mx4Args a = {};
  a.x = x; a.x_scales = (const uint8_t*)x_scales; a.ldx = ldx; a.w = (const uint8_t*)w; a.w_scales = (const uint8_t*)w_scales; a.bias = bias;
  a.out = out; a.rows = rows; a.features = a.w_rows = features; a.width = width; a.ldo = ldo;
  const dim3 grid((features + MXG_TILE - 1) / MXG_TILE, (rows + MXG_TILE - 1) / MXG_TILE);
  cudaStream_t s = (cudaStream_t)stream;
  auto kernel = x_scales ? (out_float ? mx4_product_kernel<true, MXG_F32, false> : mx4_product_kernel<true, MXG_BF16, false>)
                         : (out_float ? mx4_product_kernel<false, MXG_F32, false> : mx4_product_kernel<false, MXG_BF16, false>);
  SRB_CUDA_CALL(srb_launch(kernel, grid, dim3(256), 0, s, a));
  SRB_LAUNCH_CHECK("mx4_linear");
  return SRB_OK;
}

// The experts' products over the plan's tiles (of 64 slots): mode gated / act (rows of x through slot_row, out bfloat16 [slots, features]) or
// float (rows of x are the slots).
extern "C" int srb_mx4_experts(const void* x, long long ldx, const int* slot_row, const void* w, const void* w_scales, void* out,
                               const int* plan, int max_tiles, int experts, int features, int width, int mode, int activation,
                               float act_param, int* error_word, void* stream) {
  if (max_tiles <= 0 || features <= 0) return SRB_OK;
  if (activation < 0 || activation >= SRB_ACT_COUNT) SRB_FAIL("mx4_experts: unknown activation %d", activation);
  Mx4Args a = {};
  a.x = x; a.ldx = ldx; a.w = (const uint8_t*)w; a.w_scales = (const uint8_t*)w_scales; a.out = out; a.features = features;
  a.w_rows = mode == MXG_GATED ? 2 * features : features; a.width = width; a.ldo = features; a.activation = activation; a.act_param = act_param;
  a.plan = plan; a.slot_row = slot_row; a.experts = experts;
  const dim3 grid((features + MXG_TILE - 1) / MXG_TILE, max_tiles);
  auto kernel = mode == MXG_GATED ? mx4_product_kernel<false, MXG_GATED, true>
                : mode == MXG_ACT ? mx4_product_kernel<false, MXG_ACT, true> : mx4_product_kernel<false, MXG_F32, true>;
  SRB_CUDA_CALL(srb_launch(kernel, grid, dim3(256), 0, (cudaStream_t)stream, a));
  SRB_LAUNCH_CHECK("mx4_experts");
  return SRB_OK;
}

// out[row, :] = sum over the row's choices, in their order, of weight * y[slot, :], in 32 bits, rounded once.
__global__ void mx4_combine_kernel(const float* __restrict__ y, const int* __restrict__ entry_slot, const float* __restrict__ weights, int top,
                                   int width, __nv_bfloat16* __restrict__ out) {
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int row = blockIdx.x;
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    float sum = 0.f;
    for (int k = 0; k < top; ++k) {
      const int slot = entry_slot[(size_t)row * top + k];
      if (slot >= 0) sum = fmaf(weights[(size_t)row * top + k], y[(size_t)slot * width + i], sum);
    }
    out[(size_t)row * width + i] = __float2bfloat16_rn(sum);
  }
}
extern "C" int srb_mx4_combine(const float* y, const int* entry_slot, const float* weights, int rows, int top, int width, void* out, void* stream) {
  if (rows <= 0 || width <= 0) return SRB_OK;
  SRB_CUDA_CALL(srb_launch(mx4_combine_kernel, dim3(rows), dim3(256), 0, (cudaStream_t)stream, y, entry_slot, weights, top, width, (__nv_bfloat16*)out));
  SRB_LAUNCH_CHECK("mx4_combine");
  return SRB_OK;
}
