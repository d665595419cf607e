// Y = X W^T with W in the microscaled four-bit format of mx4.cuh, sums in 32 bits, on the block-scaled tensor cores; few rows.
//
// The weight is the M side: a block owns 128 rows of W, the N side are rows of X in four bits too (tcgen05.mma, kind mxf4).  The tensor
// cores take the entries as they are, so nothing is unpacked: turning 13 T entries a second (what the memory brings) into bfloat16 would take
// every instruction the SMs issue.  A row of bfloat16 is eight rows of four bits here (mx4.cuh, PARTS), columns of their own whose sums the
// epilogue adds: the tensor cores have time for that, a step with few rows being bound by the bytes of W.  (As two eight-bit parts, kind
// mxf8f6f4, W's entries have to stand 16 to 16 bytes in shared memory; TMA sets them so, but in pieces of 64 bytes, half of what it moves
// otherwise, and the matrices of 8 rows' experts, 64 of 2,048 x 1,408, took 66 us instead of 33.)
//
// One row the blocks turn into parts themselves, in the four warps that wait for the sums otherwise: a launch less (one row through 4,096 x 24,576 12.1 us
// instead of 13.8, 12,288 x 4,096 8.5 instead of 9.7; two rows 15.4 and 11.1 us: they keep the warps longer than the launch takes).
//
// A step is 256 entries of K.  All (else) of it comes by TMA: the rows of W and X, and both sides' scales in the tiles that mx4.cuh lays them out in,
// which the issuing thread copies to tensor memory ahead of the step's products.
//
// Two blocks an SM.  K is cut where the row tiles are fewer than the SMs: the blocks of a cluster take a part each, leave their sums in shared
// memory and add them in block order, so a result does not depend on timing.  Otherwise a block walks tiles, copying for the next one while
// the last one's sums are stored, from one of two buffers where they fit.
//
// Over experts (GROUPED) a block's rows are up to 8 slots of one expert (the plan of csrc/moe.cu), 64 rows of parts a tile.  The gated mode
// multiplies the gate rows and the up rows of 128 features into sums of their own, a feature a lane in both, and leaves act(gate) * up as parts
// again, rounded once from 32 bits, a warp's 32 features a block.
//
// Warps: 0 copies, 1 products and tensor memory, 2-5 epilogue.  Waits are bounded; one that runs out flags SRB_FLAG_WAIT_TIMEOUT.
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"
#include "mx4_rows.cuh"
#include "mx4_umma.cuh"
#include <algorithm>

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MXF_TOKENS 64            // rows of X of a tile, at most: in four bits
#define MXF_PART_TOKENS 16       // ... in parts
#define MXF_SLOTS 8              // ... over experts
#define MXF_THREADS 192
#define MXF_EPILOGUE_THREADS 128
#define MXF_W_BYTES 16384        // 128 rows x 256 entries
#define MXF_MAX_SPLITS 8         // blocks of a cluster
#define MXF_SUMS 128             // columns of tensor memory: scales lie behind
#define MXF_BF16 0     // out bfloat16 = x w^T + bias
#define MXF_F32 1      // out float
#define MXF_GATED 2    // out parts of act(x gate^T) * (x up^T), the up rows `features` behind the gate rows
#define MXF_ACT 5      // ... of act(x w^T)

struct FewArgs {
  const __nv_bfloat16* x;        // FUSED: the one row of bfloat16, of `width` entries, on a 16-byte border if x_wide
  int width, x_wide;
  const float* bias;
  void* out;
  uint8_t* out_scales;           // of parts
  size_t ldo;                    // elements; bytes of codes
  int rows, features, w_rows, k_tiles, splits;
  int tokens, columns;           // rows of X of a tile, at most; room for columns of the N side
  int ws_tiles, up_tile;         // row tiles of scales of a matrix; the one where the up rows begin
  int tiles_f, tiles_t;
  int activation;
  float act_param;
  int* error_word;
  const int* plan;               // GROUPED
  int experts;
};

template <bool GATED>
struct FewShape {
  static constexpr int SIDES = GATED ? 2 : 1;
  static constexpr int PLACE_COLUMNS = 8 * (SIDES + 1);      // of a step's scales: two tiles of 128 entries each
  static constexpr int SCALE_BYTES = 1024 * (SIDES + 1);
  static __host__ __device__ constexpr int stage_bytes(int columns) { return SIDES * MXF_W_BYTES + columns * 128; }
};

__device__ __forceinline__ float4 few_load_peer(const float* mine, unsigned rank) {
  unsigned remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}

// Sums of 16 columns: 16 rows of X, or two rows' eight parts.
template <int ROWS>
__device__ __forceinline__ void few_rows(unsigned address, float (&v)[ROWS]) {
  float sums[16];
  tmem_load_16(address, sums);
  constexpr int EACH = 16 / ROWS;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    v[r] = sums[r * EACH + EACH - 1];
#pragma unroll
    for (int p = EACH - 2; p >= 0; --p) v[r] += sums[r * EACH + p];
  }
}
// Eight lanes' words of eight half-bytes each: lane p gets half-byte p of all, that of lane i at place i.
__device__ __forceinline__ unsigned few_transpose(unsigned word, int lane) {
#pragma unroll
  for (int step = 4; step >= 1; step >>= 1) {
    const unsigned low = step == 4 ? 0x0000ffffu : step == 2 ? 0x00ff00ffu : 0x0f0f0f0fu;
    const int shift = 4 * step;
    const unsigned other = __shfl_xor_sync(0xffffffffu, word, step);
    word = lane & step ? (word & ~low) | ((other >> shift) & low) : (word & low) | ((other << shift) & ~low);
  }
  return word;
}

// 256 entries of a row of X, 8 a lane, as parts (mx4.cuh) in a stage: rows 0 .. 7 of 128 bytes, swizzled, and their scales, a byte for each 32 entries
// in each part's word of the two tiles of 128 entries.
__device__ __forceinline__ void few_make_parts(const uint4& raw, int lane, unsigned x_to, unsigned xs_to) {
  float v[8];
  mx4_unpack_bf16(raw, v);
  unsigned most = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned first = mx4_first_scale(most);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = mx4_over_first_scale(v[i], first);
#pragma unroll
  for (int part = 0; part < MX4_PARTS; ++part) {
    const unsigned row = (unsigned)part;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(x_to + row * 128 + ((((unsigned)lane >> 2) ^ row) << 4) + (lane & 3) * 4), "r"(mx4_next_part(v)) : "memory");
    if ((lane & 3) == 0)
      asm volatile("st.shared.u8 [%0], %1;" ::"r"(xs_to + (lane >> 4) * 512 + row * 16 + ((lane >> 2) & 3)), "r"(mx4_part_scale(first, part)) : "memory");
  }
}

// What a tile is, the same in every role.
struct FewTile {
  int matrix, feature0;
  int token0;                    // the first row of X (by tiles of the plan, over experts)
  int out_row0, count;
};
template <bool GROUPED>
__device__ __forceinline__ FewTile few_tile(const FewArgs& a, int item) {
  FewTile t;
  const int index = item / a.tiles_f;
  t.feature0 = item % a.tiles_f * 128;
  t.token0 = t.out_row0 = index * a.tokens;
  t.matrix = 0;
  int end = a.rows;
  if (GROUPED) {
    const int* first_slot = a.plan + 1;
    const int* tiles = first_slot + a.experts + 1;
    t.matrix = tiles[2 * index];
    t.out_row0 = tiles[2 * index + 1];
    end = first_slot[t.matrix + 1];
  }
  t.count = min(a.tokens, end - t.out_row0);
  return t;
}

template <bool PARTS, int MODE, bool GROUPED, int STAGES, bool FUSED>
__global__ void __launch_bounds__(MXF_THREADS, 2)
mx4_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_xs, const FewArgs a) {
  constexpr bool GATED = MODE == MXF_GATED, OUT_PARTS = MODE == MXF_GATED || MODE == MXF_ACT;
  constexpr int A_TOKEN = PARTS ? MX4_PARTS : 1;             // columns of a row of X
  using Shape = FewShape<GATED>;
  static_assert(STAGES * Shape::PLACE_COLUMNS <= 256 - MXF_SUMS, "a place for scales a stage");
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % a.splits;
  const int all_steps = (a.k_tiles + 1) / 2;
  const int step0 = (int)((long long)rank * all_steps / a.splits), steps = (int)((long long)(rank + 1) * all_steps / a.splits) - step0;
  const int first_item = blockIdx.x / a.splits, item_step = gridDim.x / a.splits;
  const int stage_bytes = Shape::stage_bytes(a.columns);
  const unsigned stages = smem_u32(smem), scales = stages + STAGES * stage_bytes;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), FUSED ? 2 : 1);
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
  if (!PARTS || FUSED) srb_grid_dependency_wait();
  // (With parts the kernel ahead is the one that made them, or the product ahead of this one behind it.  That kernel lets the next one start once
  // all kernels ahead of it are done, so W and the plan, which are older, may be read at once; X is awaited below.)
  const int items = (GROUPED ? a.plan[0] : a.tiles_t) * a.tiles_f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = tmem_holder;
  // a buffer of sums is `columns` for each side
  const int buffer_columns = Shape::SIDES * a.columns, buffers = buffer_columns <= MXF_SUMS / 2 ? 2 : 1;

  if (warp == 0) {
    unsigned round = 0;
    bool ok = true;
    auto load_w = [&](const FewTile& t, int s, int step) {
      const unsigned bar = smem_u32(&full_bar[s]), to = stages + s * stage_bytes, scales_to = scales + s * Shape::SCALE_BYTES;
      const int w_row = t.matrix * a.w_rows + t.feature0, ws_tile = (t.matrix * a.ws_tiles + (t.feature0 >> 7)) * a.k_tiles;
      if (elect_one()) {
        mbar_expect_tx(bar, FUSED ? Shape::SIDES * (MXF_W_BYTES + 1024) : stage_bytes + Shape::SCALE_BYTES);
        tma_load_2d(to, &map_w, bar, step * 128, w_row);
        if (GATED) tma_load_2d(to + MXF_W_BYTES, &map_w, bar, step * 128, w_row + a.features);
        tma_load_2d(scales_to, &map_ws, bar, 0, ws_tile + 2 * step);
        if (GATED) tma_load_2d(scales_to + 1024, &map_ws, bar, 0, ws_tile + a.up_tile * a.k_tiles + 2 * step);
      }
      __syncwarp();
    };
    auto load_x = [&](const FewTile& t, int s, int step) {
      const unsigned bar = smem_u32(&full_bar[s]);
      const int x_row = t.token0 * A_TOKEN;
      if (elect_one()) {
        tma_load_2d(stages + s * stage_bytes + Shape::SIDES * MXF_W_BYTES, &map_x, bar, step * 128, x_row);
        tma_load_2d(scales + s * Shape::SCALE_BYTES + 1024 * Shape::SIDES, &map_xs, bar, 0, (x_row >> 7) * a.k_tiles + 2 * step);
      }
      __syncwarp();
    };
    // the first steps' W ahead of the wait for X
    int early = 0;
    if (PARTS && !FUSED) {
      if (first_item < items) {
        const FewTile t = few_tile<GROUPED>(a, first_item);
        early = min(steps, STAGES);
        for (int i = 0; i < early; ++i) load_w(t, i, step0 + i);
      }
      srb_grid_dependency_wait();
    }
    for (int item = first_item; item < items && ok; item += item_step) {
      const FewTile t = few_tile<GROUPED>(a, item);
      for (int i = 0; i < steps; ++i, ++round) {
        const int s = (int)(round % STAGES);
        if ((int)round >= early) {
          ok = mbar_wait_warp(smem_u32(&empty_bar[s]), ((round / STAGES) & 1u) ^ 1u, &abort_flag);
          if (!ok) break;
          load_w(t, s, step0 + i);
        }
        if (!FUSED) load_x(t, s, step0 + i);
      }
    }
    if (abort_flag && round > 0) {
      // copies in flight when a wait ran out write into this block's memory: give them time to land
      const long long start = clock64();
      while (clock64() - start < 4000000ll) {}
    }
  } else if (warp == 1) {
    unsigned round = 0;
    int local = 0;
    bool ok = true;
    for (int item = first_item; item < items && ok; item += item_step, ++local) {
      const int b = local % buffers;
      const FewTile t = few_tile<GROUPED>(a, item);
      // rows of X that start in the middle of a tile of scales
      const unsigned x_shift = (unsigned)((t.token0 * A_TOKEN) & 127) >> 5;
      const unsigned idesc = mx_idesc_four(128, (t.count * A_TOKEN + 15) & ~15);
      ok = mbar_wait_warp(smem_u32(&acc_empty[b]), ((unsigned)(local / buffers) & 1u) ^ 1u, &abort_flag);
      if (!ok) break;
      tc_fence_after();
      const unsigned acc = tmem + b * buffer_columns;
      for (int i = 0; i < steps; ++i, ++round) {
        const int s = (int)(round % STAGES);
        ok = mbar_wait_warp(smem_u32(&full_bar[s]), (round / STAGES) & 1u, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        // (a place for scales a stage: who took them last is done when the stage is free)
        const unsigned at = stages + s * stage_bytes, place = tmem + MXF_SUMS + s * Shape::PLACE_COLUMNS;
        const unsigned long long w_desc = smem_descriptor(at), x_desc = smem_descriptor(at + Shape::SIDES * MXF_W_BYTES);
        const unsigned products = 2 * (step0 + i) + 1 < a.k_tiles ? 4u : 2u;
        if (elect_one()) {
          const unsigned long long from = scales_descriptor(scales + s * Shape::SCALE_BYTES);
#pragma unroll
          for (int j = 0; j < Shape::SCALE_BYTES / 512; ++j) tmem_copy_scales(place + 4 * j, from + j * (512 >> 4));
          const unsigned xs = place + 8 * Shape::SIDES + x_shift;
#pragma unroll
          for (unsigned k = 0; k < 4; ++k) {
            if (k >= products) break;
            const unsigned accumulate = (i > 0 || k > 0) ? 1u : 0u, tile = 4 * (k >> 1);
            umma_mx4(acc, w_desc + 2 * k, x_desc + 2 * k, mx_idesc_step(idesc, 2 * (k & 1)), place + tile, xs + tile, accumulate);
            if (GATED)
              umma_mx4(acc + a.columns, w_desc + (MXF_W_BYTES >> 4) + 2 * k, x_desc + 2 * k, mx_idesc_step(idesc, 2 * (k & 1)), place + 8 + tile,
                       xs + tile, accumulate);
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
      const int b = local % buffers;
      const FewTile t = few_tile<GROUPED>(a, item);
      const int feature = t.feature0 + in_tile;
      if (FUSED) {
        // the row's parts, a step's 256 entries at a time by the four warps in turn, the next ones on their way while these are made
        auto load = [&](int i) {
          const int k = (step0 + i) * 256 + lane * 8;
          uint4 raw = make_uint4(0u, 0u, 0u, 0u);
          if (a.x_wide && k + 8 <= a.width) return *reinterpret_cast<const uint4*>(a.x + k);
          unsigned short* to = reinterpret_cast<unsigned short*>(&raw);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k + j < a.width) to[j] = reinterpret_cast<const unsigned short*>(a.x)[k + j];
          return raw;
        };
        uint4 raw = make_uint4(0u, 0u, 0u, 0u), next = raw;
        bool ok = true;
        if (warp - 2 < steps) raw = load(warp - 2);
        for (int i = warp - 2; i < steps; i += 4, raw = next) {
          const unsigned round = (unsigned)(local * steps + i);
          const int s = (int)(round % STAGES);
          if (i + 4 < steps) next = load(i + 4);
          ok = mbar_wait_warp(smem_u32(&empty_bar[s]), ((round / STAGES) & 1u) ^ 1u, &abort_flag);
          if (!ok) break;
          few_make_parts(raw, lane, stages + s * stage_bytes + Shape::SIDES * MXF_W_BYTES, scales + s * Shape::SCALE_BYTES + 1024 * Shape::SIDES);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&full_bar[s]));
        }
        if (!ok) break;
      }
      if (!mbar_wait_warp(smem_u32(&acc_full[b]), (unsigned)(local / buffers) & 1u, &abort_flag)) break;
      tc_fence_after();
      const unsigned sums = lane_address + b * buffer_columns;
      const float bias = !OUT_PARTS && a.splits == 1 && a.bias && feature < a.features ? a.bias[feature] : 0.f;
      // 16 columns at a time: rows of X, or two rows' parts, added from the last on
      constexpr int AT_ONCE = 16 / A_TOKEN;
      for (int token = 0; token < t.count; token += AT_ONCE) {
        float v[AT_ONCE], up[AT_ONCE];
        few_rows<AT_ONCE>(sums + token * A_TOKEN, v);
        if (GATED) few_rows<AT_ONCE>(sums + a.columns + token * A_TOKEN, up);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (OUT_PARTS) {
            if (token + j >= t.count) break;
            float r = mx4_gated(a.activation, v[j], GATED ? up[j] : 1.0f, a.act_param);
            if (feature >= a.features) r = 0.f;              // what pads the rows of parts
            const unsigned first = mx4_first_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(r) & 0x7fffffffu));
            // part p of eight lanes' features together: lane 8 g + p gets the four bytes of features 8 g .. + 7
            const unsigned word = few_transpose(mx4_all_parts(mx4_over_first_scale(r, first)), lane);
            const int row = (t.token0 + token + j) * MX4_PARTS + (lane & 7);
            reinterpret_cast<unsigned*>(a.out)[((size_t)row * a.ldo + (feature & ~7) / 2) / 4] = word;
            if (lane < MX4_PARTS)
              a.out_scales[mx4_scale_word(row, t.feature0 >> 7, (int)(a.ldo / 64)) + quarter] = (uint8_t)mx4_part_scale(first, lane);
          } else if (a.splits > 1) {
            // (the products are done with the stages: the block has one tile)
            reinterpret_cast<float*>(smem)[(token + j) * 128 + in_tile] = v[j];
          } else if (token + j < t.count && feature < a.features) {
            const size_t at = (size_t)(t.out_row0 + token + j) * a.ldo + feature;
            if (MODE == MXF_F32) reinterpret_cast<float*>(a.out)[at] = v[j] + bias;
            else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v[j] + bias);
          }
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
      // four features of a row a thread, from all blocks at once; a block adds up a run of them (every a.splits-th in turn, a warp's 16 bytes
      // lay 128 bytes apart, all in the same banks: 48 rows of 4,096 through 4,096 features in 8 parts took 14.6 us instead of 10.7)
      const int share = (t.count * 32 + a.splits - 1) / a.splits, end = min((rank + 1) * share, t.count * 32);
      for (int i = rank * share + (int)threadIdx.x - 64; i < end; i += MXF_EPILOGUE_THREADS) {
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

template <bool PARTS, int MODE, bool GROUPED, int STAGES, bool FUSED>
static int launch_few_staged(const CUtensorMap (&maps)[4], const FewArgs& a, int blocks, cudaStream_t s) {
  using Shape = FewShape<MODE == MXF_GATED>;
  const size_t smem = 1024 + (size_t)STAGES * (Shape::stage_bytes(a.columns) + Shape::SCALE_BYTES);
  static std::atomic<int> allowed[MX4_MAX_DEVICES];
  auto kernel = mx4_few_kernel<PARTS, MODE, GROUPED, STAGES, FUSED>;
  if (const int status = mx4_allow_shared((const void*)kernel, (int)smem, allowed)) return status;
  SRB_CUDA_CALL(srb_launch_clustered(kernel, dim3(blocks), dim3(MXF_THREADS), smem, s, dim3(a.splits), maps[0], maps[1], maps[2], maps[3], a));
  return SRB_OK;
}

// x: codes [x_rows, 64 k_tiles] (parts or not) and their scales.  Stages for as much shared memory as two blocks an SM leave.
template <bool PARTS, int MODE, bool GROUPED, bool FUSED = false>
static int launch_few(const void* x, const void* x_scales, long long x_rows, const void* w, const void* w_scales, FewArgs& a, cudaStream_t s) {
  const long long matrices = std::max(a.experts, 1), w_rows = matrices * a.w_rows, ws_tiles = matrices * a.ws_tiles * a.k_tiles;
  const long long items = (long long)a.tiles_t * a.tiles_f, x_tiles = (x_rows + 127) / 128 * a.k_tiles;
  if (((uintptr_t)w | (FUSED ? 0 : (uintptr_t)x)) & 15) SRB_FAIL("mx4_few: codes must start on a 16-byte border");
  if (w_rows > 0x7fffffff || ws_tiles > 0x7fffffff || x_rows > 0x7fffffff || x_tiles > 0x7fffffff || items > 0x3fffffff)
    SRB_FAIL("mx4_few: %lld rows of weights and %lld of inputs are too many", w_rows, x_rows);
  CUtensorMap maps[4];
  if (make_bytes_map(&maps[0], w, w_rows, a.k_tiles * 64ll, 128) != SRB_OK || make_scales_map(&maps[1], w_scales, ws_tiles, 2) != SRB_OK ||
      (!FUSED && (make_bytes_map(&maps[2], x, x_rows, a.k_tiles * 64ll, a.columns) != SRB_OK || make_scales_map(&maps[3], x_scales, x_tiles, 2) != SRB_OK)))
    return SRB_ERR_INVALID;
  if (FUSED) maps[2] = maps[3] = maps[0];
  // K in parts until there is about a block an SM, or two parts where that makes two: a block costs some 3 us beside its steps (8 rows of 4,096 through
  // 4,096 features, 32 tiles, in 1, 2, 4 and 8 parts: 9.0, 7.6, 6.6 and 7.8 us; of 12,288 18.0, 12.1, 9.8 and 9.5; through 12,288 features, 96
  // tiles, in 1, 2 and 3: 9.4, 9.1 and 12.9; one row through 24,576, 192 tiles, in 1, 2 and 4: 13.8, 16.2 and 19.0)
  const long long sms = srb_sm_count(), room = 2 * sms, all_steps = (a.k_tiles + 1) / 2;
  const long long wanted = std::max(sms / items, std::min(room / items, 2ll));
  a.splits = GROUPED ? 1 : (int)std::max(1ll, std::min(std::min<long long>(wanted, MXF_MAX_SPLITS), all_steps));
  const int blocks = (int)(a.splits > 1 ? items * a.splits : std::min(items, room));
  if constexpr (MODE == MXF_GATED) return launch_few_staged<PARTS, MODE, GROUPED, 2, false>(maps, a, blocks, s);
  else if constexpr (FUSED) return launch_few_staged<PARTS, MODE, GROUPED, 5, true>(maps, a, blocks, s);
  else return a.columns <= 64 ? launch_few_staged<PARTS, MODE, GROUPED, 4, false>(maps, a, blocks, s) : launch_few_staged<PARTS, MODE, GROUPED, 3, false>(maps, a, blocks, s);
}

// ---- entries: `scratch` has srb_mx4_linear_scratch bytes (none are needed for rows in four bits) ----------------------------
extern "C" long long srb_mx4_linear_scratch(int rows, int width) {
  if (rows == 1) return 0;
  Mx4Scratch scratch = {};
  scratch.take((size_t)rows * MX4_PARTS * mx4_pitch(width));
  scratch.take((size_t)mx4_tiles(rows * MX4_PARTS) * mx4_tiles(width) * MX4_TILE_BYTES);
  return (long long)scratch.used;
}

// x: bfloat16 [rows, width], `ldx` elements apart, or (x_scales given) codes and their scales; w: codes and scales of features rows; out [rows, ldo].
extern "C" int srb_mx4_linear(const void* x, long long ldx, const void* x_scales, const void* w, const void* w_scales, const float* bias, void* out,
                              long long ldo, int rows, int features, int width, int out_float, void* scratch_memory, int* error_word, void* stream) {
  if (rows <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_linear: inner size %d must be positive", width);
  if (rows > 1 << 20) SRB_FAIL("mx4_linear: %d rows are not few", rows);
  FewArgs a = {};
  a.bias = bias; a.out = out; a.ldo = ldo; a.rows = rows; a.features = a.w_rows = features; a.k_tiles = mx4_tiles(width); a.error_word = error_word;
  a.ws_tiles = a.tiles_f = mx4_tiles(features);
  const bool parts = x_scales == nullptr;
  a.tokens = std::min(rows, parts ? MXF_PART_TOKENS : MXF_TOKENS);
  a.columns = (a.tokens * (parts ? MX4_PARTS : 1) + 15) & ~15;
  a.tiles_t = (rows + a.tokens - 1) / a.tokens;
  cudaStream_t s = (cudaStream_t)stream;
  if (!parts)
    return out_float ? launch_few<false, MXF_F32, false>(x, x_scales, rows, w, w_scales, a, s) : launch_few<false, MXF_BF16, false>(x, x_scales, rows, w, w_scales, a, s);
  if (rows == 1) {
    a.x = (const __nv_bfloat16*)x; a.width = width; a.x_wide = mx4_wide(x, 0);
    return out_float ? launch_few<true, MXF_F32, false, true>(x, nullptr, 8ll * rows, w, w_scales, a, s)
                     : launch_few<true, MXF_BF16, false, true>(x, nullptr, 8ll * rows, w, w_scales, a, s);
  }
  Mx4Scratch scratch = {(uint8_t*)scratch_memory, 0};
  uint8_t* codes = scratch.take((size_t)rows * MX4_PARTS * mx4_pitch(width));
  uint8_t* scales = scratch.take((size_t)mx4_tiles(rows * MX4_PARTS) * a.k_tiles * MX4_TILE_BYTES);
  if (const int status = mx4_launch_parts(x, ldx, rows, width, codes, scales, s)) return status;
  return out_float ? launch_few<true, MXF_F32, false>(codes, scales, 8ll * rows, w, w_scales, a, s)
                   : launch_few<true, MXF_BF16, false>(codes, scales, 8ll * rows, w, w_scales, a, s);
}

// Scratch of a call on the experts, in the order in which it is taken: rows of the slots, what is between the products, and gate/up scales with the up rows on the border of a tile, where they do not begin there.
struct FewExpertsScratch {
  uint8_t *x, *x_scales, *act, *act_scales, *up_scales;
  size_t bytes;
  FewExpertsScratch(void* memory, int max_tiles, int experts, int width, int inner, int gated) {
    Mx4Scratch s = {(uint8_t*)memory, 0};
    const size_t rows = (size_t)MXF_SLOTS * MX4_PARTS * max_tiles, row_tiles = (rows + 127) / 128;
    x = s.take(rows * mx4_pitch(width));
    x_scales = s.take(row_tiles * mx4_tiles(width) * MX4_TILE_BYTES);
    act = s.take(rows * mx4_pitch(inner));
    act_scales = s.take(row_tiles * mx4_tiles(inner) * MX4_TILE_BYTES);
    up_scales = gated && inner % 128 ? s.take(mx4_gated_scales_bytes(experts, width, 256 * mx4_tiles(inner), 1)) : nullptr;
    bytes = s.used;
  }
};
extern "C" long long srb_mx4_experts_scratch(int max_tiles, int experts, int width, int inner, int gated) {
  return (long long)FewExpertsScratch(nullptr, max_tiles, experts, width, inner, gated).bytes;
}
extern "C" int srb_mx4_experts_tile() { return MXF_SLOTS; }

// `plan` (tiles of srb_mx4_experts_tile slots, at most max_tiles) and slot_row are those of csrc/moe.cu; y float [slots, width] gets the slots' results.
extern "C" int srb_mx4_experts(const void* h, const int* plan, const int* slot_row, const void* up, const void* up_scales, const void* down,
                               const void* down_scales, float* y, int max_tiles, int slots, int experts, int width, int inner, int gated,
                               int activation, float act_param, void* scratch_memory, int* error_word, void* stream) {
  if (max_tiles <= 0) return SRB_OK;
  const Mx4ExpertsCall c = {h, plan, up, up_scales, down, down_scales, y, max_tiles, slots, experts, width, inner, gated, activation, act_param,
                            error_word, (cudaStream_t)stream};
  if (const int status = mx4_check_experts(c)) return status;
  const FewExpertsScratch scratch(scratch_memory, max_tiles, experts, width, inner, gated);
  const long long x_rows = (long long)MXF_SLOTS * MX4_PARTS * max_tiles;
  FewArgs a = {};
  a.activation = activation; a.act_param = act_param; a.error_word = error_word; a.plan = plan; a.experts = experts; a.tiles_t = max_tiles;
  a.tokens = MXF_SLOTS; a.columns = MXF_SLOTS * MX4_PARTS;
  // gate/up: into parts
  FewArgs first = a;
  first.out = scratch.act; first.out_scales = scratch.act_scales; first.features = inner; first.w_rows = gated ? 2 * inner : inner;
  first.k_tiles = mx4_tiles(width); first.tiles_f = mx4_tiles(inner); first.ldo = mx4_pitch(inner);
  first.ws_tiles = mx4_tiles(first.w_rows); first.up_tile = inner / 128;
  if (scratch.up_scales) {
    const int group = 128 * mx4_tiles(inner);
    Mx4GatedScales regroup;
    if (const int status = mx4_make_gated_scales(&regroup, up_scales, experts, inner, width, group, 2 * group, 1, 0, scratch.up_scales)) return status;
    if (const int status = mx4_launch_gated_scales(regroup, experts, plan, c.stream)) return status;
    up_scales = scratch.up_scales;
    first.ws_tiles = 2 * mx4_tiles(inner); first.up_tile = mx4_tiles(inner);
  }
  // (last ahead of the products, which read what is older than it before it is done)
  if (const int status = mx4_launch_parts_slots(h, width, plan, slot_row, experts, max_tiles, scratch.x, scratch.x_scales, c.stream)) return status;
  if (const int status = gated ? launch_few<true, MXF_GATED, true>(scratch.x, scratch.x_scales, x_rows, up, up_scales, first, c.stream)
                               : launch_few<true, MXF_ACT, true>(scratch.x, scratch.x_scales, x_rows, up, up_scales, first, c.stream)) return status;
  FewArgs second = a;
  second.out = y; second.features = second.w_rows = width; second.k_tiles = mx4_tiles(inner); second.ws_tiles = second.tiles_f = mx4_tiles(width);
  second.ldo = width;
  return launch_few<true, MXF_F32, true>(scratch.act, scratch.act_scales, x_rows, down, down_scales, second, c.stream);
}

// out bfloat16 [rows, width]: the weighted sum of every row's results.
extern "C" int srb_mx4_combine(const float* y, const int* entry_slot, const float* weights, int rows, int top, int width, void* out, void* stream) {
  if (rows <= 0 || width <= 0) return SRB_OK;
  return mx4_launch_combine(y, entry_slot, weights, rows, top, width, out, (cudaStream_t)stream);
}
