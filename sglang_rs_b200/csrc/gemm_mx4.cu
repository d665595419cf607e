// Y = X W^T with W in the microscaled four-bit format of mx4.cuh, sums in 32 bits, on the block-scaled tensor cores; few rows.
//
// The weight is the M side: a block owns 128 rows of W and up to 64 rows of X, the N side.  The tensor cores take the four-bit entries as
// they are, so nothing is unpacked: turning 13 T entries a second (what the memory brings) into bfloat16 would take every instruction the SMs
// issue.  Rows of X come as four-bit codes or as two eight-bit parts of a bfloat16 (mx4.cuh), which are columns of their own and meet in the
// epilogue.  A product step of 128 entries: the codes by TMA, which sets eight bytes to each 16 of a row in shared memory as the instruction
// wants them (by cp.async of eight bytes, 50 MB of codes took 24 us instead of LATER), and by cp.async the rows of X and both sides' scales, one
// word for each row.
//
// K is cut where the row tiles are fewer than two blocks an SM: the blocks of a cluster take a part each, leave their sums in shared memory
// and add them in block order, so a result does not depend on timing.
//
// Warps 0-3 copy (nothing waits for a copy but the products) and then store, warp 4 issues the products.  Waits are bounded; one that runs out flags SRB_FLAG_WAIT_TIMEOUT.
//
// Over experts (GROUPED) a block's rows are up to 64 slots of one expert (the plan of csrc/moe.cu).  The gated mode has 64 gate rows over the
// 64 up rows of the same features, and leaves act(gate) * up as eight-bit parts again, rounded from 32 bits, for the next product.
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"
#include "mx4_umma.cuh"
#include <algorithm>

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MXF_TOKENS 64            // rows of X of a block
#define MXF_COPY_THREADS 128
#define MXF_THREADS 160
#define MXF_A_BYTES 16384        // 128 rows x 128 entries, 16 to 16 bytes
#define MXF_BF16 0     // out bfloat16 = x w^T + bias
#define MXF_F32 1      // out float
#define MXF_GATED 2    // out two eight-bit parts of act(x gate^T) * (x up^T), the up rows `features` behind the gate rows
#define MXF_ACT 5      // ... of act(x w^T)

struct FewArgs {
  const uint8_t* x;              // codes, or the first of two parts
  const uint8_t* x_scales;
  size_t x_part, xs_part;        // bytes from the first part to the second
  const uint8_t* w_scales;
  const float* bias;
  void* out;
  uint8_t* out_scales;           // of parts
  size_t ldo;                    // elements; bytes of parts
  size_t out_part, os_part;
  int rows, features, w_rows, k_tiles, splits;
  int columns;                   // room for columns of the N side
  int activation;
  float act_param;
  int* error_word;
  const int* plan;               // GROUPED
  const int* slot_row;           // rows of x by slot, or null: the slots themselves
  int experts;
};

__device__ __forceinline__ void cp_async_8(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_4(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_16_to(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void few_copy_threads_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <bool FOUR, int MODE, bool GROUPED, int STAGES>
__global__ void __launch_bounds__(MXF_THREADS)
mx4_few_kernel(const __grid_constant__ CUtensorMap map_w, const FewArgs a) {
  constexpr bool GATED = MODE == MXF_GATED, PARTS = MODE == MXF_GATED || MODE == MXF_ACT;
  constexpr int FEATURES = GATED ? 64 : 128;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], done_bar;
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;
  __shared__ int x_row[MXF_TOKENS];

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  srb_launch_dependents();
  int matrix = 0, token0 = blockIdx.y * MXF_TOKENS, count = min(MXF_TOKENS, a.rows - token0);
  if (GROUPED) {
    srb_grid_dependency_wait();
    if ((int)blockIdx.y >= a.plan[0]) return;
    const int* tiles = a.plan + 1 + a.experts + 1;
    matrix = tiles[2 * blockIdx.y];
    token0 = tiles[2 * blockIdx.y + 1];
    count = min(MXF_TOKENS, a.plan[1 + matrix + 1] - token0);
  }
  const int part_columns = FOUR ? (count + 15) & ~15 : (count + 7) & ~7;
  const int columns = FOUR ? part_columns : 2 * part_columns;
  const int rank = blockIdx.x % a.splits, feature0 = blockIdx.x / a.splits * FEATURES;
  const int kt0 = (int)((long long)rank * a.k_tiles / a.splits), kt1 = (int)((long long)(rank + 1) * a.k_tiles / a.splits);
  const int steps = kt1 - kt0;
  const int stage_bytes = MXF_A_BYTES + a.columns * 128;
  const unsigned scales0 = smem_u32(smem) + STAGES * stage_bytes;        // per stage 512 bytes of W's and 512 of X's

  if (t == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), MXF_COPY_THREADS + 1);      // and the word that W's bytes are awaited
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    mbar_init(smem_u32(&done_bar), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) tmem_alloc(smem_u32(&tmem_holder), 256);
  if (!GROUPED) srb_grid_dependency_wait();
  if (t < MXF_TOKENS) x_row[t] = t < count ? (GROUPED && a.slot_row ? a.slot_row[token0 + t] : token0 + t) : 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = tmem_holder;
  bool ok = true;

  if (warp < 4) {
    // ---- copies: a thread has chunk t % 8 of columns t / 8 + 16 i of X, and the scales of row t of W and of column t
    const uint8_t* w_scales = a.w_scales + (size_t)matrix * mx4_tiles(a.w_rows) * a.k_tiles * MX4_TILE_BYTES;
    const int chunk = t & 7, sub = t >> 3;
    const unsigned place = (unsigned)(chunk ^ (sub & 7)) << 4;
    auto w_row = [&](int r, bool& live) {
      const int feature = feature0 + (GATED ? r & 63 : r);
      live = feature < a.features;
      return !live ? 0 : GATED && r >= 64 ? a.features + feature : feature;
    };
    bool scale_live;
    const int scale_row = w_row(t, scale_live);
    // the column of X whose scales this thread brings
    const bool second = !FOUR && t >= part_columns;
    const int x_token = second ? t - part_columns : t;
    const bool x_scale_live = t < columns && x_token < count;
    const int x_scale_row = x_scale_live ? x_row[x_token] : 0;
    const uint8_t* x_scales = a.x_scales + (second ? a.xs_part : 0);
    const size_t x_pitch = (size_t)a.k_tiles * (FOUR ? 64 : 128);
    for (int i = 0; i < steps; ++i) {
      const int s = i % STAGES, kt = kt0 + i;
      if (i >= STAGES && !mbar_wait(smem_u32(&empty_bar[s]), (unsigned)(i / STAGES - 1) & 1u, &abort_flag)) break;
      const unsigned w_to = smem_u32(smem) + s * stage_bytes, x_to = w_to + MXF_A_BYTES, scales_to = scales0 + s * 1024;
      if (warp == 0) {
        __syncwarp();
        if (elect_one()) {
          const unsigned bar = smem_u32(&full_bar[s]);
          mbar_expect_tx(bar, MXF_A_BYTES / 2);
          tma_load_2d(w_to, &map_w, bar, kt * 128, matrix * a.w_rows + feature0);
          if (GATED) tma_load_2d(w_to + MXF_A_BYTES / 2, &map_w, bar, kt * 128, matrix * a.w_rows + a.features + feature0);
        }
        __syncwarp();
      }
      cp_async_4(scales_to + lane * 16 + warp * 4, w_scales + mx4_scale_word(scale_row, kt, a.k_tiles), scale_live ? 4 : 0);
      for (int n = sub; n < columns; n += 16) {
        const bool low = !FOUR && n >= part_columns;
        const int token = low ? n - part_columns : n;
        const bool live = token < count;
        const uint8_t* src = a.x + (low ? a.x_part : 0) + (size_t)x_row[live ? token : 0] * x_pitch;
        if (FOUR) cp_async_8(x_to + n * 128 + place, src + kt * 64 + chunk * 8, live ? 8 : 0);
        else cp_async_16_to(x_to + n * 128 + place, src + kt * 128 + chunk * 16, live ? 16 : 0);
      }
      if (t < columns)
        cp_async_4(scales_to + 512 + lane * 16 + warp * 4, x_scales + mx4_scale_word(x_scale_row, kt, a.k_tiles), x_scale_live ? 4 : 0);
      copies_arrive(smem_u32(&full_bar[s]));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (abort_flag) {
      // copies by TMA in flight when a wait ran out write into this block's memory: give them time to land
      const long long start = clock64();
      while (clock64() - start < 4000000ll) {}
    }
  } else {
    // ---- products
    const unsigned idesc = mx_idesc(MX_E2M1, FOUR ? MX_E2M1 : MX_E4M3, 128, columns);
    for (int i = 0; i < steps && ok; ++i) {
      const int s = i % STAGES;
      ok = mbar_wait_warp(smem_u32(&full_bar[s]), (unsigned)(i / STAGES) & 1u, &abort_flag);
      if (!ok) break;
      fence_proxy_async_shared();
      tc_fence_after();
      const unsigned w_at = smem_u32(smem) + s * stage_bytes;
      const unsigned long long a_desc = smem_descriptor(w_at), b_desc = smem_descriptor(w_at + MXF_A_BYTES);
      const unsigned sa = tmem + 128 + 8 * s, sb = sa + 4;
      if (elect_one()) {
        tmem_copy_scales(sa, scales_descriptor(scales0 + s * 1024));
        tmem_copy_scales(sb, scales_descriptor(scales0 + s * 1024 + 512));
#pragma unroll
        for (unsigned k = 0; k < 4; ++k)
          umma_mx8(tmem, a_desc + 2 * k, b_desc + 2 * k, mx_idesc_step(idesc, k), sa, sb, (i > 0 || k > 0) ? 1u : 0u);
        umma_commit(smem_u32(&empty_bar[s]));
        if (i == steps - 1) umma_commit(smem_u32(&done_bar));
      }
      __syncwarp();
    }
  }

  // ---- epilogue: warp w has lanes 32 w .. + 31 of tensor memory, a row of W a lane, and all columns
  float* shared = reinterpret_cast<float*>(smem);            // the stages are done with
  if (warp < 4) {
    mbar_wait_warp(smem_u32(&done_bar), 0u, &abort_flag);
    few_copy_threads_sync();
    ok = *reinterpret_cast<volatile int*>(&abort_flag) == 0;  // the same in every warp
    tc_fence_after();
  }
  const unsigned lane_address = tmem + ((unsigned)(warp * 32) << 16);
  auto eight = [&](int token, float (&v)[8]) {
    tmem_load_8(lane_address + token, v);
    if (!FOUR) {
      float low[8];
      tmem_load_8(lane_address + part_columns + token, low);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += low[j];
    }
  };
  auto store = [&](int token, int feature, float v) {
    if (a.bias) v += a.bias[feature];
    const size_t at = (size_t)(token0 + token) * a.ldo + feature;
    if (MODE == MXF_F32) reinterpret_cast<float*>(a.out)[at] = v;
    else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  };
  if (PARTS) {
    if (warp < 4 && ok) {
      if (GATED) {
        if (warp >= 2) {
          for (int token = 0; token < count; token += 8) {
            float v[8];
            eight(token, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) shared[(token + j) * 64 + (t & 63)] = v[j];
          }
        }
        few_copy_threads_sync();
      }
      if (!GATED || warp < 2) {
        const int feature = feature0 + t;
        for (int token = 0; token < count; token += 8) {
          float v[8];
          eight(token, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (token + j >= count) break;
            float r = srb_gated<true>(a.activation, v[j], GATED ? shared[(token + j) * 64 + t] : 1.0f, a.act_param);
            if (feature >= a.features) r = 0.f;              // behind the rows of W: the part that pads the parts' rows
            const unsigned high = mx8_scale_high(__reduce_max_sync(0xffffffffu, __float_as_uint(r) & 0x7fffffffu)), low = mx8_scale_low(high);
            unsigned high_byte, low_byte;
            mx8_split(r, 0.f, high, low, high_byte, low_byte);
            uint8_t* dst = reinterpret_cast<uint8_t*>(a.out) + (size_t)(token0 + token + j) * a.ldo + feature;
            dst[0] = (uint8_t)high_byte;
            dst[a.out_part] = (uint8_t)low_byte;
            if (lane == 0) {
              uint8_t* scale = a.out_scales + mx4_scale_word(token0 + token + j, feature >> 7, (int)(a.ldo / 128)) + ((feature >> 5) & 3);
              scale[0] = (uint8_t)high;
              scale[a.os_part] = (uint8_t)low;
            }
          }
        }
      }
    }
  } else if (a.splits == 1) {
    if (warp < 4 && ok) {
      const int feature = feature0 + t;
      for (int token = 0; token < count; token += 8) {
        float v[8];
        eight(token, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (token + j < count && feature < a.features) store(token + j, feature, v[j]);
      }
    }
  } else {
    if (warp < 4 && ok) {
      for (int token = 0; token < count; token += 8) {
        float v[8];
        eight(token, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) shared[(token + j) * 128 + t] = v[j];
      }
    }
    srb_cluster_sync();
    if (warp < 4 && ok) {
      const int feature = feature0 + t;
      for (int token = rank; token < count; token += a.splits) {
        float sum = 0.f;
        for (int r = 0; r < a.splits; ++r) sum += srb_load_peer_shared(shared + token * 128 + t, r);
        if (feature < a.features) store(token, feature, sum);
      }
    }
    srb_cluster_sync();                                      // nobody leaves while its sums may still be read
  }
  tc_fence_before();
  __syncthreads();
  if (t == 0 && abort_flag) atomicOr(a.error_word, SRB_FLAG_WAIT_TIMEOUT);
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <bool FOUR, int MODE, bool GROUPED, int STAGES>
static int launch_few_staged(const CUtensorMap& map_w, const FewArgs& a, int tiles_f, int tiles_t, cudaStream_t s) {
  const size_t smem = 1024 + (size_t)STAGES * (MXF_A_BYTES + a.columns * 128 + 1024);
  auto kernel = mx4_few_kernel<FOUR, MODE, GROUPED, STAGES>;
  SRB_CUDA_CALL(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  SRB_CUDA_CALL(srb_launch_clustered(kernel, dim3(tiles_f * a.splits, tiles_t), dim3(MXF_THREADS), smem, s, dim3(a.splits), map_w, a));
  SRB_LAUNCH_CHECK("mx4_few");
  return SRB_OK;
}

// Two blocks an SM: stages for as much shared memory as that leaves.
template <bool FOUR, int MODE, bool GROUPED>
static int launch_few(const void* w, FewArgs& a, int tokens, int tiles_f, int tiles_t, cudaStream_t s) {
  CUtensorMap map_w;
  const long long w_rows = (long long)std::max(a.experts, 1) * a.w_rows;
  if ((uintptr_t)w & 31) SRB_FAIL("mx4_few: codes must start on a 32-byte border");
  if (w_rows > 0x7fffffff) SRB_FAIL("mx4_few: %lld rows of weights are too many", w_rows);
  if (make_codes_map(&map_w, w, w_rows, a.k_tiles, MODE == MXF_GATED ? 64 : 128) != SRB_OK) return SRB_ERR_INVALID;
  tokens = std::min(tokens, MXF_TOKENS);
  a.columns = FOUR ? (tokens + 15) & ~15 : 2 * ((tokens + 7) & ~7);
  if (tiles_t > 65535) SRB_FAIL("mx4_few: %d tiles of rows are too many", tiles_t);
  return a.columns <= 32 ? launch_few_staged<FOUR, MODE, GROUPED, 5>(map_w, a, tiles_f, tiles_t, s)
         : a.columns <= 64 ? launch_few_staged<FOUR, MODE, GROUPED, 4>(map_w, a, tiles_f, tiles_t, s)
                           : launch_few_staged<FOUR, MODE, GROUPED, 3>(map_w, a, tiles_f, tiles_t, s);
}

// K in parts until there are about two blocks an SM, at least two steps each.
static int few_splits(long long tiles, int k_tiles) {
  const long long wanted = 2ll * srb_sm_count() / std::max(tiles, 1ll);
  return (int)std::max(1ll, std::min(std::min(wanted, 8ll), (long long)k_tiles / 2));
}

// x: codes [rows, 64 k_tiles] with their scales (`four`), or parts [2, rows, 128 k_tiles] with theirs; w: codes [features, 64 k_tiles]; out
// [rows, ldo].
extern "C" int srb_mx4_linear(const void* x, const void* x_scales, int four, const void* w, const void* w_scales, const float* bias,
                              void* out, long long ldo, int rows, int features, int width, int out_float, int* error_word, void* stream) {
  if (rows <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_linear: inner size %d must be positive", width);
  FewArgs a = {};
  a.x = (const uint8_t*)x; a.x_scales = (const uint8_t*)x_scales; a.w_scales = (const uint8_t*)w_scales; a.bias = bias;
  a.out = out; a.ldo = ldo; a.rows = rows; a.features = a.w_rows = features; a.k_tiles = mx4_tiles(width); a.error_word = error_word;
  a.x_part = (size_t)rows * a.k_tiles * 128; a.xs_part = (size_t)mx4_tiles(rows) * a.k_tiles * MX4_TILE_BYTES;
  const int tiles_f = mx4_tiles(features), tiles_t = (rows + MXF_TOKENS - 1) / MXF_TOKENS;
  a.splits = few_splits((long long)tiles_f * tiles_t, a.k_tiles);
  cudaStream_t s = (cudaStream_t)stream;
  if (four)
    return out_float ? launch_few<true, MXF_F32, false>(w, a, rows, tiles_f, tiles_t, s) : launch_few<true, MXF_BF16, false>(w, a, rows, tiles_f, tiles_t, s);
  return out_float ? launch_few<false, MXF_F32, false>(w, a, rows, tiles_f, tiles_t, s) : launch_few<false, MXF_BF16, false>(w, a, rows, tiles_f, tiles_t, s);
}

// The experts' products over the plan's tiles (of 64 slots).  x: parts [2, x_rows, 128 k_tiles] and their scales; rows by `slot_row`, or the
// slots themselves (null).  Mode gated / act: out parts [2, slots, 128 ceil(features / 128)], out_scales theirs; float: out [slots, features].
extern "C" int srb_mx4_experts(const void* x, const void* x_scales, int x_rows, const int* slot_row, const void* w, const void* w_scales,
                               void* out, void* out_scales, const int* plan, int max_tiles, int slots, int experts, int features, int width,
                               int mode, int activation, float act_param, int* error_word, void* stream) {
  if (max_tiles <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_experts: inner size %d must be positive", width);
  if (activation < 0 || activation >= SRB_ACT_COUNT) SRB_FAIL("mx4_experts: unknown activation %d", activation);
  if (mode != MXF_F32 && mode != MXF_GATED && mode != MXF_ACT) SRB_FAIL("mx4_experts: mode %d is not float, gated or activated", mode);
  FewArgs a = {};
  a.x = (const uint8_t*)x; a.x_scales = (const uint8_t*)x_scales; a.w_scales = (const uint8_t*)w_scales; a.out = out;
  a.out_scales = (uint8_t*)out_scales; a.rows = slots; a.features = features; a.w_rows = mode == MXF_GATED ? 2 * features : features;
  a.k_tiles = mx4_tiles(width); a.activation = activation; a.act_param = act_param; a.error_word = error_word;
  a.x_part = (size_t)x_rows * a.k_tiles * 128; a.xs_part = (size_t)mx4_tiles(x_rows) * a.k_tiles * MX4_TILE_BYTES;
  a.plan = plan; a.slot_row = slot_row; a.experts = experts; a.splits = 1;
  cudaStream_t s = (cudaStream_t)stream;
  const int out_tiles = mx4_tiles(features);
  if (mode == MXF_F32) {
    a.ldo = features;
    return launch_few<false, MXF_F32, true>(w, a, slots, out_tiles, max_tiles, s);
  }
  a.ldo = (size_t)out_tiles * 128;
  a.out_part = (size_t)slots * a.ldo; a.os_part = (size_t)mx4_tiles(slots) * out_tiles * MX4_TILE_BYTES;
  if (mode == MXF_GATED) return launch_few<false, MXF_GATED, true>(w, a, slots, 2 * out_tiles, max_tiles, s);
  return launch_few<false, MXF_ACT, true>(w, a, slots, out_tiles, max_tiles, s);
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
