// Y = X W^T with W in the microscaled four-bit format of mx4.cuh, sums in 32 bits, on the block-scaled tensor cores; few rows.
//
// The weight is the M side: a block owns 128 rows of W and up to 64 rows of X, the N side.  The tensor cores take the four-bit entries as
// they are, so nothing is unpacked: turning 13 T entries a second (what the memory brings) into bfloat16 would take every instruction the SMs
// issue.  Rows of X come as four-bit codes or as the two eight-bit parts of a bfloat16 (mx4.cuh), each multiplied into the same sums.
//
// A step is 128 entries of K.  All of it comes by TMA: the codes, set eight bytes to each 16 as kind mxf8f6f4 wants them, the rows of X, and
// both sides' scales in the tiles that mx4.cuh lays them out in, which the issuing thread copies to tensor memory ahead of the step's products.
// (With cp.async for the scales and for X a step took 700 cycles however many were in flight: the fence that ordinary writes need ahead of the
// products stands in the products' way.)
//
// Two blocks an SM.  K is cut where the row tiles are fewer than that: the blocks of a cluster take a part each, leave their sums in shared
// memory and add them in block order, so a result does not depend on timing.  Otherwise a block walks tiles, copying for the next one while
// the last one's sums, in one of two buffers, are stored.
//
// Over experts (GROUPED) a block's rows are up to 32 slots of one expert (the plan of csrc/moe.cu), X and the parts that the first product
// leaves having room for 64 rows a tile: scales of a product may begin at an even column of tensor memory alone (an odd one faults), that is at a
// multiple of 64 rows.  The gated mode multiplies the gate rows and the up rows of 128 features into sums of their own, a feature
// a lane in both, and leaves act(gate) * up as eight-bit parts, rounded once from 32 bits, a warp's 32 features a block.
//
// Warps: 0 copies, 1 products and tensor memory, 2-5 epilogue.  Waits are bounded; one that runs out flags SRB_FLAG_WAIT_TIMEOUT.
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"
#include "mx4_umma.cuh"
#include <algorithm>

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MXF_TOKENS 64            // rows of X of a tile, at most
#define MXF_SLOTS 32             // ... over experts, at most
#define MXF_ROOM 64              // ... and rows that a tile has room for
#define MXF_THREADS 192
#define MXF_EPILOGUE_THREADS 128
#define MXF_W_BYTES 16384        // 128 rows x 128 entries, 16 to 16 bytes
#define MXF_MAX_SPLITS 8         // blocks of a cluster
#define MXF_PLACES 4             // of a step's scales in tensor memory
#define MXF_BF16 0     // out bfloat16 = x w^T + bias
#define MXF_F32 1      // out float
#define MXF_GATED 2    // out two eight-bit parts of act(x gate^T) * (x up^T), the up rows `features` behind the gate rows
#define MXF_ACT 5      // ... of act(x w^T)

struct FewArgs {
  const float* bias;
  void* out;
  uint8_t* out_scales;           // of parts
  size_t ldo;                    // elements; bytes of parts
  size_t out_part, os_part;
  int rows, features, w_rows, k_tiles, splits;
  int columns;                   // of the N side: rows of X of a tile, up to a multiple of 16
  int x_lo_row, xs_lo_tile;      // where the second part's rows and tiles of scales begin
  int ws_tiles, up_tile;         // row tiles of scales of a matrix; the one where the up rows begin
  int tiles_f, tiles_t;
  int activation;
  float act_param;
  int* error_word;
  const int* plan;               // GROUPED
  int experts, tile_slots;
};

template <bool FOUR, bool GATED>
struct FewShape {
  static constexpr int PARTS = FOUR ? 1 : 2, SIDES = GATED ? 2 : 1;
  static constexpr int PLACE_COLUMNS = 4 * (SIDES + PARTS);
  static constexpr int SCALE_BYTES = 512 * (SIDES + PARTS);
  static __host__ __device__ constexpr int stage_bytes(int columns) { return SIDES * MXF_W_BYTES + PARTS * columns * 128; }
  // what the barrier counts: codes without the gaps
  static __host__ __device__ constexpr int tx_bytes(int columns) { return SIDES * MXF_W_BYTES / 2 + (FOUR ? columns * 64 : 2 * columns * 128) + SCALE_BYTES; }
};

__device__ __forceinline__ float4 few_load_peer(const float* mine, unsigned rank) {
  unsigned remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}

// What a tile is, the same in every role.
struct FewTile {
  int matrix, feature0;
  int x_row0;                    // the first row of X (with room for MXF_ROOM a tile, over experts)
  int out_row0, count;
};
template <bool GROUPED>
__device__ __forceinline__ FewTile few_tile(const FewArgs& a, int item) {
  FewTile t;
  if (GROUPED) {
    const int* first_slot = a.plan + 1;
    const int* tiles = first_slot + a.experts + 1;
    const int index = item / a.tiles_f;
    t.matrix = tiles[2 * index];
    t.out_row0 = tiles[2 * index + 1];
    t.count = min(a.tile_slots, first_slot[t.matrix + 1] - t.out_row0);
    t.x_row0 = index * MXF_ROOM;
    t.feature0 = item % a.tiles_f * 128;
  } else {
    t.matrix = 0;
    t.x_row0 = t.out_row0 = item / a.tiles_f * MXF_TOKENS;
    t.count = min(MXF_TOKENS, a.rows - t.out_row0);
    t.feature0 = item % a.tiles_f * 128;
  }
  return t;
}

template <bool FOUR, int MODE, bool GROUPED, int STAGES>
__global__ void __launch_bounds__(MXF_THREADS, 2)
mx4_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_xs, const FewArgs a) {
  constexpr bool GATED = MODE == MXF_GATED, PARTS = MODE == MXF_GATED || MODE == MXF_ACT;
  using Shape = FewShape<FOUR, GATED>;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % a.splits;
  const int kt0 = (int)((long long)rank * a.k_tiles / a.splits), steps = (int)((long long)(rank + 1) * a.k_tiles / a.splits) - kt0;
  const int first_item = blockIdx.x / a.splits, item_step = gridDim.x / a.splits;
  const int stage_bytes = Shape::stage_bytes(a.columns);
  const unsigned stages = smem_u32(smem), scales = stages + STAGES * stage_bytes;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), MXF_EPILOGUE_THREADS / 32);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_holder), 256);
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int items = (GROUPED ? a.plan[0] : a.tiles_t) * a.tiles_f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = tmem_holder;
  // sums: a buffer is `columns` for each side; scales lie behind 128 columns
  const int buffer_columns = Shape::SIDES * a.columns;

  if (warp == 0) {
    unsigned round = 0;
    bool ok = true;
    for (int item = first_item; item < items && ok; item += item_step) {
      const FewTile t = few_tile<GROUPED>(a, item);
      const int w_row = t.matrix * a.w_rows + t.feature0;
      const int ws_tile = (t.matrix * a.ws_tiles + (t.feature0 >> 7)) * a.k_tiles, xs_tile = (t.x_row0 >> 7) * a.k_tiles;
      for (int i = 0; i < steps; ++i, ++round) {
        const int s = (int)(round % STAGES), kt = kt0 + i;
        ok = mbar_wait_warp(smem_u32(&empty_bar[s]), ((round / STAGES) & 1u) ^ 1u, &abort_flag);
        if (!ok) break;
        const unsigned bar = smem_u32(&full_bar[s]), to = stages + s * stage_bytes, scales_to = scales + s * Shape::SCALE_BYTES;
        if (elect_one()) {
          mbar_expect_tx(bar, Shape::tx_bytes(a.columns));
          tma_load_2d(to, &map_w, bar, kt * 128, w_row);
          tma_load_2d(scales_to, &map_ws, bar, 0, ws_tile + kt);
          if (GATED) {
            tma_load_2d(to + MXF_W_BYTES, &map_w, bar, kt * 128, w_row + a.features);
            tma_load_2d(scales_to + 512, &map_ws, bar, 0, ws_tile + a.up_tile * a.k_tiles + kt);
          }
          const unsigned x_to = to + Shape::SIDES * MXF_W_BYTES, xs_to = scales_to + 512 * Shape::SIDES;
          tma_load_2d(x_to, &map_x, bar, kt * 128, t.x_row0);
          tma_load_2d(xs_to, &map_xs, bar, 0, xs_tile + kt);
          if (!FOUR) {
            tma_load_2d(x_to + a.columns * 128, &map_x, bar, kt * 128, a.x_lo_row + t.x_row0);
            tma_load_2d(xs_to + 512, &map_xs, bar, 0, a.xs_lo_tile + xs_tile + kt);
          }
        }
        __syncwarp();
      }
    }
    if (abort_flag && round > 0) {
      // copies in flight when a wait ran out write into this block's memory: give them time to land
      const long long start = clock64();
      while (clock64() - start < 4000000ll) {}
    }
  } else if (warp == 1) {
    const unsigned idesc = mx_idesc(MX_E2M1, FOUR ? MX_E2M1 : MX_E4M3, 128, a.columns);
    unsigned round = 0;
    int local = 0;
    bool ok = true;
    for (int item = first_item; item < items && ok; item += item_step, ++local) {
      const int b = local & 1;
      // rows of X that start in the middle of a tile of scales
      const unsigned x_shift = (unsigned)(few_tile<GROUPED>(a, item).x_row0 & 127) >> 5;
      ok = mbar_wait_warp(smem_u32(&acc_empty[b]), (((unsigned)local >> 1) & 1u) ^ 1u, &abort_flag);
      if (!ok) break;
      tc_fence_after();
      const unsigned acc = tmem + b * buffer_columns;
      for (int i = 0; i < steps; ++i, ++round) {
        const int s = (int)(round % STAGES);
        ok = mbar_wait_warp(smem_u32(&full_bar[s]), (round / STAGES) & 1u, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        const unsigned at = stages + s * stage_bytes, place = tmem + 128 + (round % MXF_PLACES) * Shape::PLACE_COLUMNS;
        const unsigned long long w_desc = smem_descriptor(at), x_desc = smem_descriptor(at + Shape::SIDES * MXF_W_BYTES);
        const unsigned long long x_lo = (unsigned long long)(a.columns * 128 >> 4);
        if (elect_one()) {
          const unsigned long long from = scales_descriptor(scales + s * Shape::SCALE_BYTES);
#pragma unroll
          for (int j = 0; j < Shape::SCALE_BYTES / 512; ++j) tmem_copy_scales(place + 4 * j, from + j * (512 >> 4));
          const unsigned xs = place + 4 * Shape::SIDES + x_shift;
#pragma unroll
          for (int part = 0; part < Shape::PARTS; ++part)
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
              const unsigned accumulate = (i > 0 || part > 0 || k > 0) ? 1u : 0u;
              umma_mx8(acc, w_desc + 2 * k, x_desc + part * x_lo + 2 * k, mx_idesc_step(idesc, k), place, xs + 4 * part, accumulate);
              if (GATED)
                umma_mx8(acc + a.columns, w_desc + (MXF_W_BYTES >> 4) + 2 * k, x_desc + part * x_lo + 2 * k, mx_idesc_step(idesc, k),
                         place + 4, xs + 4 * part, accumulate);
            }
          umma_commit(smem_u32(&empty_bar[s]));
          if (i == steps - 1) umma_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    }
  } else {
    // ---- epilogue: warp w has lanes 32 (w % 4) .. + 31 of tensor memory, a feature a lane, and all columns
    const int quarter = warp & 3, in_tile = quarter * 32 + lane;
    const unsigned lane_address = tmem + ((unsigned)(quarter * 32) << 16);
    int local = 0;
    for (int item = first_item; item < items; item += item_step, ++local) {
      const int b = local & 1;
      const FewTile t = few_tile<GROUPED>(a, item);
      const int feature = t.feature0 + in_tile;
      if (!mbar_wait_warp(smem_u32(&acc_full[b]), ((unsigned)local >> 1) & 1u, &abort_flag)) break;
      tc_fence_after();
      const unsigned sums = lane_address + b * buffer_columns;
      const float bias = !PARTS && a.splits == 1 && a.bias && feature < a.features ? a.bias[feature] : 0.f;
      for (int token = 0; token < t.count; token += 8) {
        float v[8];
        tmem_load_8(sums + token, v);
        if (PARTS) {
          float up[8];
          if (GATED) tmem_load_8(sums + a.columns + token, up);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (token + j >= t.count) break;
            float r = srb_gated<true>(a.activation, v[j], GATED ? up[j] : 1.0f, a.act_param);
            if (feature >= a.features) r = 0.f;              // the part that pads the parts' rows
            const unsigned high = mx8_scale_high(__reduce_max_sync(0xffffffffu, __float_as_uint(r) & 0x7fffffffu)), low = mx8_scale_low(high);
            unsigned high_byte, low_byte;
            mx8_split(r, 0.f, high, low, high_byte, low_byte);
            const int row = t.x_row0 + token + j;
            uint8_t* dst = reinterpret_cast<uint8_t*>(a.out) + (size_t)row * a.ldo + feature;
            dst[0] = (uint8_t)high_byte;
            dst[a.out_part] = (uint8_t)low_byte;
            if (lane == 0) {
              uint8_t* scale = a.out_scales + mx4_scale_word(row, feature >> 7, (int)(a.ldo / 128)) + quarter;
              scale[0] = (uint8_t)high;
              scale[a.os_part] = (uint8_t)low;
            }
          }
        } else if (a.splits == 1) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (token + j < t.count && feature < a.features) {
              const size_t at = (size_t)(t.out_row0 + token + j) * a.ldo + feature;
              if (MODE == MXF_F32) reinterpret_cast<float*>(a.out)[at] = v[j] + bias;
              else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v[j] + bias);
            }
        } else {
          // (the products are done with the stages: the block has one tile)
#pragma unroll
          for (int j = 0; j < 8; ++j) reinterpret_cast<float*>(smem)[(token + j) * 128 + in_tile] = v[j];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
    }
  }
  if (a.splits > 1) {
    __syncwarp();
    srb_cluster_sync();
    const FewTile t = few_tile<GROUPED>(a, first_item);
    if (warp >= 2 && abort_flag == 0) {
      // four features of a row a thread, from all blocks at once
      for (int i = rank + a.splits * ((int)threadIdx.x - 64); i < t.count * 32; i += a.splits * MXF_EPILOGUE_THREADS) {
        float4 part[MXF_MAX_SPLITS];
#pragma unroll
        for (int r = 0; r < MXF_MAX_SPLITS; ++r)
          if (r < a.splits) part[r] = few_load_peer(reinterpret_cast<float*>(smem) + 4 * i, r);
        float4 sum = part[0];
#pragma unroll
        for (int r = 1; r < MXF_MAX_SPLITS; ++r)
          if (r < a.splits) sum = make_float4(sum.x + part[r].x, sum.y + part[r].y, sum.z + part[r].z, sum.w + part[r].w);
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        const int feature = t.feature0 + 4 * (i & 31);
        const size_t at = (size_t)(t.out_row0 + (i >> 5)) * a.ldo + feature;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (feature + j < a.features) {
            const float r = v[j] + (a.bias ? a.bias[feature + j] : 0.f);
            if (MODE == MXF_F32) reinterpret_cast<float*>(a.out)[at + j] = r;
            else reinterpret_cast<__nv_bfloat16*>(a.out)[at + j] = __float2bfloat16_rn(r);
          }
      }
    }
    __syncwarp();
    srb_cluster_sync();                                      // nobody leaves while its sums may still be read
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) atomicOr(a.error_word, SRB_FLAG_WAIT_TIMEOUT);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <bool FOUR, int MODE, bool GROUPED, int STAGES>
static int launch_few_staged(const CUtensorMap (&maps)[4], const FewArgs& a, int blocks, cudaStream_t s) {
  using Shape = FewShape<FOUR, MODE == MXF_GATED>;
  const size_t smem = 1024 + (size_t)STAGES * (Shape::stage_bytes(a.columns) + Shape::SCALE_BYTES);
  auto kernel = mx4_few_kernel<FOUR, MODE, GROUPED, STAGES>;
  SRB_CUDA_CALL(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  SRB_CUDA_CALL(srb_launch_clustered(kernel, dim3(blocks), dim3(MXF_THREADS), smem, s, dim3(a.splits), maps[0], maps[1], maps[2], maps[3], a));
  SRB_LAUNCH_CHECK("mx4_few");
  return SRB_OK;
}

// x_rows, x_scale_tiles: of all parts.  Stages for as much shared memory as two blocks an SM leave.
template <bool FOUR, int MODE, bool GROUPED>
static int launch_few(const void* x, const void* x_scales, long long x_rows, long long x_scale_tiles, const void* w, const void* w_scales, FewArgs& a,
                      cudaStream_t s) {
  const long long matrices = std::max(a.experts, 1), w_rows = matrices * a.w_rows, ws_tiles = matrices * a.ws_tiles * a.k_tiles;
  const long long items = (long long)a.tiles_t * a.tiles_f;
  if (((uintptr_t)w | (uintptr_t)x) & 31) SRB_FAIL("mx4_few: codes and rows must start on a 32-byte border");
  if (w_rows > 0x7fffffff || ws_tiles > 0x7fffffff || x_rows > 0x7fffffff || x_scale_tiles > 0x7fffffff || items > 0x3fffffff)
    SRB_FAIL("mx4_few: %lld rows of weights and %lld of inputs are too many", w_rows, x_rows);
  CUtensorMap maps[4];
  if (make_codes_map(&maps[0], w, w_rows, a.k_tiles, 128) != SRB_OK || make_scales_map(&maps[1], w_scales, ws_tiles, 1) != SRB_OK ||
      (FOUR ? make_codes_map(&maps[2], x, x_rows, a.k_tiles, a.columns) : make_bytes_map(&maps[2], x, x_rows, a.k_tiles * 128ll, a.columns)) != SRB_OK ||
      make_scales_map(&maps[3], x_scales, x_scale_tiles, 1) != SRB_OK)
    return SRB_ERR_INVALID;
  // K in parts until there are about two blocks an SM, at least two steps each
  const long long room = 2ll * srb_sm_count();
  a.splits = GROUPED ? 1 : (int)std::max(1ll, std::min(std::min<long long>(room / items, MXF_MAX_SPLITS), (long long)a.k_tiles / 2));
  const int blocks = (int)(a.splits > 1 ? items * a.splits : std::min(items, room));
  if (MODE == MXF_GATED) return a.columns <= 16 ? launch_few_staged<FOUR, MODE, GROUPED, 3>(maps, a, blocks, s) : launch_few_staged<FOUR, MODE, GROUPED, 2>(maps, a, blocks, s);
  return a.columns * (FOUR ? 1 : 2) <= 32 ? launch_few_staged<FOUR, MODE, GROUPED, 5>(maps, a, blocks, s)
         : a.columns * (FOUR ? 1 : 2) <= 64 ? launch_few_staged<FOUR, MODE, GROUPED, 4>(maps, a, blocks, s)
                                            : launch_few_staged<FOUR, MODE, GROUPED, 3>(maps, a, blocks, s);
}

// x: codes [rows, 64 k_tiles] with their scales (`four`), or parts [2, rows, 128 k_tiles] with theirs; w: codes [features, 64 k_tiles]; out
// [rows, ldo].
extern "C" int srb_mx4_linear(const void* x, const void* x_scales, int four, const void* w, const void* w_scales, const float* bias,
                              void* out, long long ldo, int rows, int features, int width, int out_float, int* error_word, void* stream) {
  if (rows <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_linear: inner size %d must be positive", width);
  FewArgs a = {};
  a.bias = bias; a.out = out; a.ldo = ldo; a.rows = rows; a.features = a.w_rows = features; a.k_tiles = mx4_tiles(width); a.error_word = error_word;
  a.x_lo_row = rows; a.xs_lo_tile = mx4_tiles(rows) * a.k_tiles; a.ws_tiles = a.tiles_f = mx4_tiles(features);
  a.tiles_t = (rows + MXF_TOKENS - 1) / MXF_TOKENS;
  a.columns = (std::min(rows, MXF_TOKENS) + 15) & ~15;
  const long long parts = four ? 1 : 2, x_rows = parts * rows, xs_tiles = parts * a.xs_lo_tile;
  cudaStream_t s = (cudaStream_t)stream;
  if (four)
    return out_float ? launch_few<true, MXF_F32, false>(x, x_scales, x_rows, xs_tiles, w, w_scales, a, s)
                     : launch_few<true, MXF_BF16, false>(x, x_scales, x_rows, xs_tiles, w, w_scales, a, s);
  return out_float ? launch_few<false, MXF_F32, false>(x, x_scales, x_rows, xs_tiles, w, w_scales, a, s)
                   : launch_few<false, MXF_BF16, false>(x, x_scales, x_rows, xs_tiles, w, w_scales, a, s);
}

// The experts' products over the plan's tiles of `tile_slots` (32 at most) slots.  x: parts [2, 64 max_tiles, 128 k_tiles] and their scales, 64 rows a
// tile.  Mode gated / act: out parts [2, 64 max_tiles, 128 ceil(features / 128)], out_scales theirs; float: out [slots, features].  The
// gated mode: `up_scale_row` is the row of w_scales' tiles where the up rows begin, a multiple of 128; `scale_rows` the rows that they hold a matrix.
extern "C" int srb_mx4_experts(const void* x, const void* x_scales, const void* w, const void* w_scales, int scale_rows, int up_scale_row, void* out,
                               void* out_scales, const int* plan, int tile_slots, int max_tiles, int experts, int features, int width, int mode,
                               int activation, float act_param, int* error_word, void* stream) {
  if (max_tiles <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_experts: inner size %d must be positive", width);
  if (tile_slots != 16 && tile_slots != MXF_SLOTS) SRB_FAIL("mx4_experts: tiles of %d slots are not 16 or %d", tile_slots, MXF_SLOTS);
  if (activation < 0 || activation >= SRB_ACT_COUNT) SRB_FAIL("mx4_experts: unknown activation %d", activation);
  if (mode != MXF_F32 && mode != MXF_GATED && mode != MXF_ACT) SRB_FAIL("mx4_experts: mode %d is not float, gated or activated", mode);
  if (mode == MXF_GATED && up_scale_row % 128) SRB_FAIL("mx4_experts: scales of up rows begin at row %d, no multiple of 128", up_scale_row);
  FewArgs a = {};
  a.out = out; a.out_scales = (uint8_t*)out_scales; a.features = features; a.w_rows = mode == MXF_GATED ? 2 * features : features;
  a.k_tiles = mx4_tiles(width); a.activation = activation; a.act_param = act_param; a.error_word = error_word;
  a.ws_tiles = mx4_tiles(scale_rows); a.up_tile = up_scale_row >> 7;
  a.plan = plan; a.experts = experts; a.tile_slots = a.columns = tile_slots;
  a.tiles_f = mx4_tiles(features); a.tiles_t = max_tiles;
  const long long rows = (long long)MXF_ROOM * max_tiles, tiles = (rows + 127) / 128;
  a.x_lo_row = (int)rows; a.xs_lo_tile = (int)tiles * a.k_tiles;
  cudaStream_t s = (cudaStream_t)stream;
  if (mode == MXF_F32) {
    a.ldo = features;
    return launch_few<false, MXF_F32, true>(x, x_scales, 2 * rows, 2 * tiles * a.k_tiles, w, w_scales, a, s);
  }
  a.ldo = (size_t)a.tiles_f * 128;
  a.out_part = (size_t)rows * a.ldo; a.os_part = (size_t)tiles * a.tiles_f * MX4_TILE_BYTES;
  if (mode == MXF_GATED) return launch_few<false, MXF_GATED, true>(x, x_scales, 2 * rows, 2 * tiles * a.k_tiles, w, w_scales, a, s);
  return launch_few<false, MXF_ACT, true>(x, x_scales, 2 * rows, 2 * tiles * a.k_tiles, w, w_scales, a, s);
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
