// Y = X W^T with W in the microscaled four-bit format of mx4.cuh for many rows: tiles of 256 rows of X x 192 rows of W on pairs of CTAs
// (tcgen05.mma.cta_group::2 with block scales), in a persistent loop.
//
// Two kinds of rows.  FOUR: X in four bits too; both operands and their scales come by TMA as they lie, a step is 256 entries, four
// products of kind mxf4 (64 entries each, four times bfloat16's rate).  Otherwise X is the two eight-bit parts of a bfloat16 (mx4.cuh): a
// step is 128 entries, four products of kind mxf8f6f4 for each part into the same sums (each at twice bfloat16's rate); they want the codes of W
// eight bytes to each 16, as TMA sets them.  Nothing is unpacked in either.
//
// CTA r of a pair has 128 rows of X (the M side) and 96 rows of W (half of the N side) in shared memory, and in tensor memory two
// buffers of 192 columns of sums for its rows of X, a row a lane, beside 128 columns of scales (256 columns of sums twice would leave none).  Scales
// go from shared to tensor memory ahead of a step's products, in the same queue: products wait for the copies issued ahead of them, copies not for the
// products, so each stage has a place for scales of its own, which is free when the stage is.
//
// Over experts (GROUPED) a tile is up to 256 slots of one expert (the plan of csrc/moe.cu); X and the parts that the gated mode leaves have room
// for 256 rows a tile, so that a tile's scales are whole tiles.  Gated: the even CTA brings gate rows, the odd one the up rows of the same 96 features,
// whose scales come regrouped (mx4_gated_scales: 96 and 96 rows are no whole tiles; a word a row by cp.async instead kept the tensor cores
// waiting, 296 us instead of some 215 for the gate/up of 12,288 slots, 64 experts of 2,048 x 1,408, as the epilogue then was; those of experts with more
// than 48 slots take 145 us now, the tensor pipe active 0.73 of them).
//
// Bound by the tensor cores under the chip's power limit: 2,048 rows of bfloat16 through 4,096 x 24,576 in 262 to 267 us for some milliseconds (1,560
// TFLOP/s of the product, twice that of the parts' products: 0.95 of the library's bfloat16 rate), 310 again and again.  Both operands in four bits by
// what L2 brings, 10.3 TB/s: 95 to 97 us and 113 again and again (4,300 TFLOP/s), 8 us of it the rows' quantising.  Without the copies of scales
// it takes no less; a sixth stage with five places for scales, each awaited ahead of its next copies, 109 to 116: tensor memory has no columns for a
// sixth place.  Tiles of 384 rows of W in one buffer, which bring X half as often, took the same (260, 93 with six stages): nothing is multiplied
// while they are stored.
//
// Warps: 0 TMA, 1 products (even CTA) and tensor memory, 2-13 epilogue: a quarter of the lanes and a third of the columns each.  Waits are
// bounded; one that runs out flags SRB_FLAG_WAIT_TIMEOUT.
#include "common.cuh"
#include "activations.cuh"
#include "mx4.cuh"
#include "mx4_rows.cuh"
#include "mx4_umma.cuh"
#include <algorithm>

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define MXP_ROWS 128             // rows of X of a CTA
#define MXP_TILE 256             // ... of a pair
#define MXP_N 192                // rows of W of a pair
#define MXP_HALF 96
#define MXP_EPILOGUE_WARPS 12
#define MXP_BOX_BYTES 2048       // a warp's piece of the output: 32 rows x 64 bytes, swizzled
#define MXP_A_BYTES (MXP_ROWS * 128)
#define MXP_B_BYTES (MXP_HALF * 128)
#define MXP_SUMS 384             // columns of tensor memory: scales lie behind
#define MXP_BF16 0
#define MXP_F32 1
#define MXP_GATED 2
#define MXP_ACT 5

template <bool FOUR> struct PairShape {
  static constexpr int STAGES = FOUR ? 5 : 4;
  static constexpr int PARTS = FOUR ? 1 : 2;
  static constexpr int B_AT = PARTS * MXP_A_BYTES;
  static constexpr int XS_AT = B_AT + MXP_B_BYTES;           // scales of X: two column tiles, or a tile of each part
  static constexpr int WS_AT = XS_AT + 1024;                 // of W: two row tiles of each column tile, or 192 rows in order
  static constexpr int STAGE_BYTES = WS_AT + (FOUR ? 2048 : 1024);
  static constexpr int TMA_BYTES = FOUR ? STAGE_BYTES : 2 * MXP_A_BYTES + MXP_B_BYTES / 2 + 2048;    // what the barrier counts: codes without the gaps
  static constexpr int THREADS = 32 * (2 + MXP_EPILOGUE_WARPS);
  static constexpr int PLACE_COLUMNS = FOUR ? 24 : 16;       // of scales of a step
};

struct PairMx4Args {
  const float* bias;
  void* out;
  uint8_t* out_scales;           // of parts
  size_t ldo;                    // elements; bytes of parts
  size_t out_part, os_part;
  int rows, features, w_rows, k_tiles;
  int x_lo_row, xs_lo_tile;      // where the second part's rows and tiles of scales begin
  int ws_tiles;                  // row tiles of scales of a matrix
  int tiles_t, tiles_f;
  int by_element;                // rows of the result that do not start on 16-byte borders: no TMA
  int activation;
  float act_param;
  int* error_word;
  const int* plan;               // GROUPED
  int experts;
};

__device__ __forceinline__ void pair_tmem_alloc(unsigned holder) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "r"(512) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(unsigned address) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(512) : "memory");
}
// arrives on the barrier at this offset in both CTAs once the products and copies issued so far are done
__device__ __forceinline__ void pair_commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((unsigned short)3) : "memory");
}
// a copy whose bytes count on the even CTA's barrier (bit 24 of a shared address names the odd CTA)
__device__ __forceinline__ void pair_tma_load(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void arrive_at(unsigned bar, unsigned rank) {
  asm volatile("{\n.reg .b32 remote;\nmapa.shared::cluster.u32 remote, %0, %1;\n"
               "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [remote];\n}\n" ::"r"(bar), "r"(rank) : "memory");
}
__device__ __forceinline__ void pair_tma_store(const CUtensorMap* map, unsigned src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(src), "r"(x), "r"(y) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void pair_stores_have_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_16(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ unsigned two_bf16(float low, float high) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const unsigned*>(&v);
}

// A warp's box (`live` rows of 64 bytes, swizzled) to rows that start anywhere: the lanes take neighbouring entries, a row of 32 bfloat16 at a time or two
// of 16 floats (2,048 rows of bfloat16 through 4,096 x 24,575: 274 us, 24,576 by TMA 266; both in four bits 97 and 92, through 512 x 24,575 54 and 41).
template <bool FLOAT>
__device__ __forceinline__ void pair_store_elements(const PairMx4Args& a, unsigned box, int first, int live, int feature, int lane) {
  constexpr int WIDTH = FLOAT ? 16 : 32, BYTES = FLOAT ? 4 : 2;
  const int column = lane % WIDTH;
  if (feature + column >= a.features) return;
#pragma unroll 4
  for (int r = lane / WIDTH; r < live; r += 32 / WIDTH) {
    const unsigned from = box + r * 64 + ((((unsigned)column * BYTES >> 4) ^ ((unsigned)(r >> 1) & 3u)) << 4) + (column * BYTES & 15);
    const size_t at = (size_t)(first + r) * a.ldo + feature + column;
    if (FLOAT) {
      unsigned v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
      reinterpret_cast<unsigned*>(a.out)[at] = v;
    } else {
      unsigned short v;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
      reinterpret_cast<unsigned short*>(a.out)[at] = v;
    }
  }
}

// What a tile is, the same in every role of both CTAs.
struct PairMx4Tile {
  int feature0;                  // the first output feature
  int x_row0;                    // the first row of X (of the padded ones, over experts)
  int out_row0, limit;           // the first row (or slot) of the result, and where the tile's rows end
  int matrix;
};
template <int MODE, bool GROUPED>
__device__ __forceinline__ PairMx4Tile pair_mx4_tile(const PairMx4Args& a, int tile) {
  constexpr int FEATURES = MODE == MXP_GATED ? MXP_HALF : MXP_N;
  PairMx4Tile t;
  if (GROUPED) {
    // the features of a row tile follow one another: its rows stay in L2, and an expert's weights are streamed once
    const int* first_slot = a.plan + 1;
    const int* tiles = first_slot + a.experts + 1;
    const int rt = tile / a.tiles_f;
    t.matrix = tiles[2 * rt];
    t.feature0 = (tile % a.tiles_f) * FEATURES;
    t.x_row0 = rt * MXP_TILE;
    t.out_row0 = tiles[2 * rt + 1];
    t.limit = min(t.out_row0 + MXP_TILE, first_slot[t.matrix + 1]);
  } else {
    t.matrix = 0;
    t.feature0 = tile / a.tiles_t * FEATURES;
    t.x_row0 = t.out_row0 = tile % a.tiles_t * MXP_TILE;
    t.limit = a.rows;
  }
  return t;
}

template <bool FOUR, int MODE, bool GROUPED>
__global__ void __launch_bounds__(PairShape<FOUR>::THREADS, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_out, const PairMx4Args a) {
  using Shape = PairShape<FOUR>;
  constexpr int STAGES = Shape::STAGES;
  static_assert(STAGES * Shape::PLACE_COLUMNS <= 512 - MXP_SUMS, "a place for scales a stage");
  constexpr bool GATED = MODE == MXP_GATED, PARTS = MODE == MXP_GATED || MODE == MXP_ACT;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = srb_cluster_rank();                  // 0: the CTA that issues the products
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int steps = FOUR ? (a.k_tiles + 1) / 2 : a.k_tiles;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 2 * MXP_EPILOGUE_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) pair_tmem_alloc(smem_u32(&tmem_holder));
  tc_fence_before();
  srb_cluster_sync();
  tc_fence_after();
  const unsigned tmem = tmem_holder;
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int num_tiles = GROUPED ? a.plan[0] * a.tiles_f : a.tiles_t * a.tiles_f;

  if (warp == 0) {
    // ---- TMA: each CTA its own halves; the bytes count on the even CTA's barrier
    int issued = 0;
    unsigned round = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      const PairMx4Tile t = pair_mx4_tile<MODE, GROUPED>(a, tile);
      const int x_row = t.x_row0 + (int)rank * MXP_ROWS, xs_tile = (x_row >> 7) * a.k_tiles;
      const int w_row = t.matrix * a.w_rows + t.feature0 + (int)rank * (GATED ? a.features : MXP_HALF);
      // (the gated mode's scales are in groups of 96 gate and 96 up rows, two tiles each)
      const int ws_tile = (t.matrix * a.ws_tiles + (GATED ? t.feature0 / MXP_HALF * 2 : t.feature0 >> 7)) * a.k_tiles;
      for (int i = 0; i < steps && ok; ++i, ++round) {
        const int s = (int)(round % STAGES);
        ok = mbar_wait_warp(smem_u32(&empty_bar[s]), ((round / STAGES) & 1u) ^ 1u, &abort_flag);
        if (!ok) break;
        const unsigned bar = smem_u32(&full_bar[s]), stage = smem_u32(smem) + s * Shape::STAGE_BYTES;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(bar, 2 * Shape::TMA_BYTES);
          pair_tma_load(stage, &map_x, bar, i * 128, x_row);
          if (FOUR) {
            pair_tma_load(stage + Shape::B_AT, &map_w, bar, i * 128, w_row);
            pair_tma_load(stage + Shape::XS_AT, &map_xs, bar, 0, xs_tile + 2 * i);
            pair_tma_load(stage + Shape::WS_AT, &map_ws, bar, 0, ws_tile + 2 * i);
            pair_tma_load(stage + Shape::WS_AT + 1024, &map_ws, bar, 0, ws_tile + a.k_tiles + 2 * i);
          } else {
            pair_tma_load(stage + MXP_A_BYTES, &map_x, bar, i * 128, a.x_lo_row + x_row);
            pair_tma_load(stage + Shape::XS_AT, &map_xs, bar, 0, xs_tile + i);
            pair_tma_load(stage + Shape::B_AT, &map_w, bar, i * 128, w_row);
            pair_tma_load(stage + Shape::XS_AT + 512, &map_xs, bar, 0, a.xs_lo_tile + xs_tile + i);
            pair_tma_load(stage + Shape::WS_AT, &map_ws, bar, 0, ws_tile + i);
            pair_tma_load(stage + Shape::WS_AT + 512, &map_ws, bar, 0, ws_tile + a.k_tiles + i);
          }
        }
        ++issued;
      }
    }
    // copies in flight when a wait ran out write into this CTA's memory: give them time to land
    if (abort_flag && issued > 0) {
      const long long start = clock64();
      while (clock64() - start < 4000000ll) {}
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- products of the pair
      const unsigned idesc = FOUR ? mx_idesc_four(2 * MXP_ROWS, MXP_N) : mx_idesc(MX_E4M3, MX_E2M1, 2 * MXP_ROWS, MXP_N);
      unsigned round = 0;
      int local = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int b = local & 1;
        ok = mbar_wait_warp_cluster(smem_u32(&acc_empty[b]), (((unsigned)local >> 1) & 1u) ^ 1u, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        const unsigned acc = tmem + b * MXP_N;
        // a tile of W that starts in the middle of a tile of scales
        const unsigned shift = !GATED ? (unsigned)(pair_mx4_tile<MODE, GROUPED>(a, tile).feature0 & 127) >> 5 : 0u;
        for (int i = 0; i < steps && ok; ++i, ++round) {
          const int s = (int)(round % STAGES);
          ok = mbar_wait_warp_cluster(smem_u32(&full_bar[s]), (round / STAGES) & 1u, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          const unsigned stage = smem_u32(smem) + s * Shape::STAGE_BYTES;
          // (a place for scales a stage: who took them last is done when the stage is free)
          const unsigned place = tmem + MXP_SUMS + s * Shape::PLACE_COLUMNS;
          const unsigned long long a_desc = smem_descriptor(stage), b_desc = smem_descriptor(stage + Shape::B_AT);
          if (elect_one()) {
            const unsigned long long xs = scales_descriptor(stage + Shape::XS_AT), ws = scales_descriptor(stage + Shape::WS_AT);
            tmem_copy_scales_pair(place, xs);
            tmem_copy_scales_pair(place + 4, xs + (512 >> 4));
            if (FOUR) {
              // rows of the first row tile, of the second; this column tile, the next
              tmem_copy_scales_pair(place + 8, ws);
              tmem_copy_scales_pair(place + 12, ws + (1024 >> 4));
              tmem_copy_scales_pair(place + 16, ws + (512 >> 4));
              tmem_copy_scales_pair(place + 20, ws + (1536 >> 4));
              const unsigned products = 2 * i + 1 < a.k_tiles ? 4u : 2u;
#pragma unroll
              for (unsigned k = 0; k < 4; ++k)
                if (k < products)
                  umma_mx4_pair(acc, a_desc + 2 * k, b_desc + 2 * k, mx_idesc_step(idesc, 2 * (k & 1)), place + 4 * (k >> 1),
                                place + 8 + 8 * (k >> 1) + shift, (i > 0 || k > 0) ? 1u : 0u);
            } else {
              tmem_copy_scales_pair(place + 8, ws);
              tmem_copy_scales_pair(place + 12, ws + (512 >> 4));
#pragma unroll
              for (unsigned k = 0; k < 8; ++k)
                umma_mx8_pair(acc, a_desc + (k >> 2) * (MXP_A_BYTES >> 4) + 2 * (k & 3), b_desc + 2 * (k & 3), mx_idesc_step(idesc, k & 3),
                              place + 4 * (k >> 2), place + 8 + shift, (i > 0 || k > 0) ? 1u : 0u);
            }
            pair_commit(smem_u32(&empty_bar[s]));
            if (i == steps - 1) pair_commit(smem_u32(&acc_full[b]));
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ---- epilogue: warp w has lanes 32 * (w % 4) .. + 31 of its CTA's tensor memory, a row of X a lane, and a third of the columns
    const int quarter = warp & 3, third = (warp - 2) >> 2;
    const unsigned lane_address = tmem + ((unsigned)(quarter * 32) << 16);
    const unsigned box = smem_u32(smem) + STAGES * Shape::STAGE_BYTES + (warp - 2) * MXP_BOX_BYTES;
    int local = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++local) {
      const int b = local & 1;
      const PairMx4Tile t = pair_mx4_tile<MODE, GROUPED>(a, tile);
      const int first = t.out_row0 + (int)rank * MXP_ROWS + quarter * 32, live = min(t.limit - first, 32);
      if (!mbar_wait_warp(smem_u32(&acc_full[b]), ((unsigned)local >> 1) & 1u, &abort_flag)) break;
      tc_fence_after();
      const unsigned sums = lane_address + b * MXP_N;
      if (live > 0) {
        if (PARTS) {
          // a lane's 32 features are a block of the next product's rows
#pragma unroll 1
          for (int part = 0; part < (GATED ? 1 : 2); ++part) {
            const int column = GATED ? third * 32 : third * 64 + part * 32, feature = t.feature0 + column;
            if (feature >= (int)a.ldo) continue;
            float v[32];
            tmem_load_32(sums + column, v);
            if (GATED) {
              float up[32];
              tmem_load_32(sums + MXP_HALF + column, up);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = mx4_gated(a.activation, lane < live ? v[j] : 1.0f, up[j], a.act_param);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = mx4_gated(a.activation, lane < live ? v[j] : 1.0f, 1.0f, a.act_param);
            }
            if (feature + 32 > a.features) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (feature + j >= a.features) v[j] = 0.f;   // the part that pads the parts' rows
            }
            if (lane < live) {
              unsigned most = 0u;
#pragma unroll
              for (int j = 0; j < 32; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
              const unsigned high = mx8_scale_high(most), low = mx8_scale_low(high);
              unsigned h[8], l[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                unsigned h0, l0, h1, l1;
                mx8_split(v[4 * j], v[4 * j + 1], high, low, h0, l0);
                mx8_split(v[4 * j + 2], v[4 * j + 3], high, low, h1, l1);
                h[j] = h0 | h1 << 16;
                l[j] = l0 | l1 << 16;
              }
              const int row = t.x_row0 + (int)rank * MXP_ROWS + quarter * 32 + lane;
              uint8_t* dst = reinterpret_cast<uint8_t*>(a.out) + (size_t)row * a.ldo + feature;
              reinterpret_cast<uint4*>(dst)[0] = make_uint4(h[0], h[1], h[2], h[3]);
              reinterpret_cast<uint4*>(dst)[1] = make_uint4(h[4], h[5], h[6], h[7]);
              reinterpret_cast<uint4*>(dst + a.out_part)[0] = make_uint4(l[0], l[1], l[2], l[3]);
              reinterpret_cast<uint4*>(dst + a.out_part)[1] = make_uint4(l[4], l[5], l[6], l[7]);
              uint8_t* scale = a.out_scales + mx4_scale_word(row, feature >> 7, (int)(a.ldo / 128)) + ((feature >> 5) & 3);
              scale[0] = (uint8_t)high;
              scale[a.os_part] = (uint8_t)low;
            }
          }
        } else {
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {
            const int column = third * 64 + part * 32, feature = t.feature0 + column;
            if (feature >= a.features) continue;
            float v[32];
            tmem_load_32(sums + column, v);
            if (a.bias) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] += feature + j < a.features ? __ldg(a.bias + feature + j) : 0.f;
            }
            if (GROUPED && live < 32) {
              // the rows behind the expert's last slot belong to the next one
              float* dst = reinterpret_cast<float*>(a.out) + (size_t)(first + lane) * a.ldo + feature;
              if (lane < live) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (feature + j < a.features) dst[j] = v[j];
              }
              continue;
            }
            // 64 bytes of a row: 32 features in bfloat16, 16 in float; a 16-byte piece goes where the store's 64-byte swizzle wants it
            const unsigned row = box + lane * 64;
            const unsigned turn = (unsigned)(lane >> 1) & 3u;
#pragma unroll
            for (int half = 0; half < (MODE == MXP_F32 ? 2 : 1); ++half) {
              if (lane == 0) pair_stores_have_read();
              __syncwarp();
#pragma unroll
              for (unsigned i = 0; i < 4; ++i) {
                if (MODE == MXP_F32) {
                  const float* q = v + 16 * half + 4 * i;
                  store_16(row + ((i ^ turn) << 4), __float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3]));
                } else {
                  const float* q = v + 8 * i;
                  store_16(row + ((i ^ turn) << 4), two_bf16(q[0], q[1]), two_bf16(q[2], q[3]), two_bf16(q[4], q[5]), two_bf16(q[6], q[7]));
                }
              }
              if (!GROUPED && a.by_element) {
                __syncwarp();
                pair_store_elements<MODE == MXP_F32>(a, box, first, live, feature + 16 * half, lane);
                continue;
              }
              fence_proxy_async_shared();
              __syncwarp();
              if (lane == 0 && feature + 16 * half < a.features) pair_tma_store(&map_out, box, feature + 16 * half, first);
            }
          }
        }
      }
      // the buffer is free for the tile after next
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(smem_u32(&acc_empty[b]), 0);
    }
    if (lane == 0) pair_stores_have_read();                  // before this block's shared memory goes
    tc_fence_before();
  }
  __syncwarp();
  srb_cluster_sync();                                        // nobody leaves while the other CTA may still signal or read
  if (threadIdx.x == 0 && abort_flag) atomicOr(a.error_word, SRB_FLAG_WAIT_TIMEOUT);
  if (warp == 1) {
    tc_fence_after();
    pair_tmem_dealloc(tmem);
  }
}

// ------------------------------------------------------------------------------- host side
template <bool FOUR, int MODE, bool GROUPED>
static int launch_pair(const CUtensorMap (&maps)[5], const PairMx4Args& a, int max_tiles, cudaStream_t s) {
  using Shape = PairShape<FOUR>;
  const int pairs = std::max(1, std::min(srb_sm_count() / 2, max_tiles));
  const size_t smem = (size_t)Shape::STAGES * Shape::STAGE_BYTES + MXP_EPILOGUE_WARPS * MXP_BOX_BYTES + 1024;
  static std::atomic<int> allowed[MX4_MAX_DEVICES];
  auto kernel = mx4_pair_kernel<FOUR, MODE, GROUPED>;
  if (const int status = mx4_allow_shared((const void*)kernel, (int)smem, allowed)) return status;
  SRB_CUDA_CALL(srb_launch_clustered(kernel, dim3(2 * pairs), dim3(Shape::THREADS), smem, s, dim3(2), maps[0], maps[1], maps[2], maps[3], maps[4], a));
  return SRB_OK;
}

// ---- entries, as those of gemm_mx4.cu --------------------------------------------------------------------------------
extern "C" long long srb_mx4_linear_pair_scratch(int rows, int width) {
  Mx4Scratch scratch = {};
  scratch.take(2 * (size_t)rows * mx4_tiles(width) * 128);
  scratch.take(2 * (size_t)mx4_tiles(rows) * mx4_tiles(width) * MX4_TILE_BYTES);
  return (long long)scratch.used;
}

// out's rows are `ldo` elements apart.
extern "C" int srb_mx4_linear_pair(const void* x, long long ldx, const void* x_scales, const void* w, const void* w_scales, const float* bias, void* out,
                                   long long ldo, int rows, int features, int width, int out_float, void* scratch_memory, int* error_word, void* stream) {
  if (rows <= 0 || features <= 0) return SRB_OK;
  if (width <= 0) SRB_FAIL("mx4_linear_pair: inner size %d must be positive", width);
  if (((uintptr_t)w & 31) || (x_scales && ((uintptr_t)x & 31))) SRB_FAIL("mx4_linear_pair: codes must start on 32-byte borders");
  PairMx4Args a = {};
  a.bias = bias; a.out = out; a.ldo = ldo; a.rows = rows; a.features = a.w_rows = features; a.k_tiles = mx4_tiles(width); a.error_word = error_word;
  a.by_element = ((uintptr_t)out & 15) != 0 || ldo * (out_float ? 4 : 2) % 16 != 0;
  a.tiles_t = (rows + MXP_TILE - 1) / MXP_TILE; a.tiles_f = (features + MXP_N - 1) / MXP_N; a.ws_tiles = mx4_tiles(features);
  const long long row_tiles = mx4_tiles(rows), tiles = (long long)a.tiles_t * a.tiles_f, scale_tiles = 2 * row_tiles * a.k_tiles;
  if (tiles > 0x3fffffff || 2ll * row_tiles * 128 > 0x7fffffff || scale_tiles > 0x7fffffff || (long long)a.ws_tiles * a.k_tiles > 0x7fffffff)
    SRB_FAIL("mx4_linear_pair: %d rows x %d features of %d are too many", rows, features, width);
  a.x_lo_row = rows; a.xs_lo_tile = (int)(row_tiles * a.k_tiles);
  cudaStream_t s = (cudaStream_t)stream;
  const bool four = x_scales != nullptr;
  if (!four) {
    Mx4Scratch scratch = {(uint8_t*)scratch_memory, 0};
    uint8_t* parts = scratch.take(2 * (size_t)rows * a.k_tiles * 128);
    uint8_t* scales = scratch.take((size_t)scale_tiles * MX4_TILE_BYTES);
    if (const int status = mx4_launch_split(x, ldx, rows, width, parts, scales, s)) return status;
    x = parts; x_scales = scales;
  }
  CUtensorMap maps[5];
  if (make_bytes_map(&maps[0], x, four ? rows : 2ll * rows, a.k_tiles * (four ? 64 : 128), MXP_ROWS) != SRB_OK ||
      make_scales_map(&maps[1], x_scales, four ? scale_tiles / 2 : scale_tiles, four ? 2 : 1) != SRB_OK ||
      (four ? make_bytes_map(&maps[2], w, features, a.k_tiles * 64, MXP_HALF) : make_codes_map(&maps[2], w, features, a.k_tiles, MXP_HALF)) != SRB_OK ||
      make_scales_map(&maps[3], w_scales, (long long)a.ws_tiles * a.k_tiles, four ? 2 : 1) != SRB_OK)
    return SRB_ERR_INVALID;
  maps[4] = maps[0];
  if (!a.by_element && make_map(&maps[4], out_float ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, rows, features,
                                ldo * (out_float ? 4 : 2), 32, out_float ? 16 : 32, CU_TENSOR_MAP_SWIZZLE_64B) != SRB_OK)
    return SRB_ERR_INVALID;
  if (four) return out_float ? launch_pair<true, MXP_F32, false>(maps, a, (int)tiles, s) : launch_pair<true, MXP_BF16, false>(maps, a, (int)tiles, s);
  return out_float ? launch_pair<false, MXP_F32, false>(maps, a, (int)tiles, s) : launch_pair<false, MXP_BF16, false>(maps, a, (int)tiles, s);
}

// One of the experts' products over the plan's tiles.  x: parts [2, 256 max_tiles, 128 k_tiles] and their scales, 256 rows a tile.  Gated / activated:
// out parts of that form, out_scales theirs; float: out [slots, features], rows on 16-byte borders.  The gated mode's w_scales are in
// groups of 96 gate and 96 up rows in the room of 256.
static int pair_experts_product(int mode, const Mx4ExpertsCall& c, const uint8_t* x, const uint8_t* x_scales, const void* w, const void* w_scales, void* out,
                                uint8_t* out_scales, int features, int width) {
  PairMx4Args a = {};
  a.out = out; a.out_scales = out_scales; a.rows = c.slots; a.features = features; a.w_rows = mode == MXP_GATED ? 2 * features : features;
  a.k_tiles = mx4_tiles(width); a.activation = c.activation; a.act_param = c.act_param; a.error_word = c.error_word; a.plan = c.plan; a.experts = c.experts;
  const long long rows = (long long)MXP_TILE * c.max_tiles;
  const int out_tiles = mx4_tiles(features), covered = mode == MXP_F32 ? features : 128 * out_tiles, per_tile = mode == MXP_GATED ? MXP_HALF : MXP_N;
  a.x_lo_row = (int)rows; a.xs_lo_tile = 2 * c.max_tiles * a.k_tiles;
  a.tiles_f = (covered + per_tile - 1) / per_tile;
  a.ws_tiles = mode == MXP_GATED ? 2 * a.tiles_f : out_tiles;
  a.ldo = covered;
  a.out_part = (size_t)rows * a.ldo; a.os_part = (size_t)2 * c.max_tiles * out_tiles * MX4_TILE_BYTES;
  const long long w_rows = (long long)c.experts * a.w_rows, ws_tiles = (long long)c.experts * a.ws_tiles * a.k_tiles;
  if (2 * rows > 0x7fffffff || w_rows > 0x7fffffff || ws_tiles > 0x7fffffff || 4ll * c.max_tiles * a.k_tiles > 0x7fffffff ||
      (long long)c.max_tiles * a.tiles_f > 0x3fffffff)
    SRB_FAIL("four-bit experts: %d tiles of rows, %lld rows of weights are too many", c.max_tiles, w_rows);
  CUtensorMap maps[5];
  if (make_bytes_map(&maps[0], x, 2 * rows, a.k_tiles * 128, MXP_ROWS) != SRB_OK ||
      make_scales_map(&maps[1], x_scales, 4ll * c.max_tiles * a.k_tiles, 1) != SRB_OK || make_codes_map(&maps[2], w, w_rows, a.k_tiles, MXP_HALF) != SRB_OK ||
      make_scales_map(&maps[3], w_scales, ws_tiles, 1) != SRB_OK)
    return SRB_ERR_INVALID;
  maps[4] = maps[0];
  if (mode == MXP_F32 && make_map(&maps[4], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, out, a.rows, features, features * 4ll, 32, 16, CU_TENSOR_MAP_SWIZZLE_64B) != SRB_OK)
    return SRB_ERR_INVALID;
  const int tiles = c.max_tiles * a.tiles_f;
  if (mode == MXP_F32) return launch_pair<false, MXP_F32, true>(maps, a, tiles, c.stream);
  if (mode == MXP_GATED) return launch_pair<false, MXP_GATED, true>(maps, a, tiles, c.stream);
  return launch_pair<false, MXP_ACT, true>(maps, a, tiles, c.stream);
}

struct PairExpertsScratch {
  uint8_t *x, *x_scales, *act, *act_scales, *up_scales;
  size_t bytes;
  int groups;                    // of 96 gate and 96 up rows
  PairExpertsScratch(void* memory, int max_tiles, int experts, int width, int inner, int gated) {
    Mx4Scratch s = {(uint8_t*)memory, 0};
    const size_t rows = 2 * (size_t)MXP_TILE * max_tiles;
    groups = (128 * mx4_tiles(inner) + MXP_HALF - 1) / MXP_HALF;
    x = s.take(rows * mx4_tiles(width) * 128);
    x_scales = s.take(rows / 128 * mx4_tiles(width) * MX4_TILE_BYTES);
    act = s.take(rows * mx4_tiles(inner) * 128);
    act_scales = s.take(rows / 128 * mx4_tiles(inner) * MX4_TILE_BYTES);
    up_scales = gated ? s.take(mx4_gated_scales_bytes(experts, width, 256, groups)) : nullptr;
    bytes = s.used;
  }
};
extern "C" long long srb_mx4_experts_pair_scratch(int max_tiles, int experts, int width, int inner, int gated) {
  return (long long)PairExpertsScratch(nullptr, max_tiles, experts, width, inner, gated).bytes;
}
extern "C" int srb_mx4_experts_pair_tile() { return MXP_TILE; }

// As srb_mx4_experts, from the slots of the `rows` rows' choices, `top` each, instead of the slots' rows; experts of up to `few_slots` slots
// have no tile in the plan; width is a multiple of 4.
extern "C" int srb_mx4_experts_pair(const void* h, const int* plan, const int* entry_slot, const void* up, const void* up_scales, const void* down,
                                    const void* down_scales, float* y, int max_tiles, int rows, int top, int few_slots, int experts, int width, int inner, int gated,
                                    int activation, float act_param, void* scratch_memory, int* error_word, void* stream) {
  if (max_tiles <= 0) return SRB_OK;
  const Mx4ExpertsCall c = {h, plan, up, up_scales, down, down_scales, y, max_tiles, rows * top, experts, width, inner, gated, activation, act_param,
                            error_word, (cudaStream_t)stream};
  if (const int status = mx4_check_experts(c)) return status;
  if (width % 4) SRB_FAIL("mx4_experts_pair: width %d is no multiple of 4", width);
  const PairExpertsScratch scratch(scratch_memory, max_tiles, experts, width, inner, gated);
  Mx4GatedScales regroup = {};
  if (gated) {
    if (const int status = mx4_make_gated_scales(&regroup, up_scales, experts, inner, width, MXP_HALF, 256, scratch.groups, few_slots, scratch.up_scales)) return status;
    up_scales = scratch.up_scales;
  }
  if (const int status = mx4_launch_split_slots(h, rows, width, plan, entry_slot, top, experts, max_tiles, scratch.x, scratch.x_scales, regroup, gated ? experts : 0,
                                                c.stream)) return status;
  if (const int status = pair_experts_product(gated ? MXP_GATED : MXP_ACT, c, scratch.x, scratch.x_scales, up, up_scales, scratch.act, scratch.act_scales,
                                              inner, width)) return status;
  return pair_experts_product(MXP_F32, c, scratch.act, scratch.act_scales, down, down_scales, y, nullptr, width, inner);
}

// A plan's experts between the two kernels: those with up to `limit` slots get tiles of `few_tile` slots in `few`, the others of 256 in `many`.  Both
// are plans like the first: number of tiles, first slots, (expert, first slot) of every tile.  One block, an expert a thread.
__global__ void __launch_bounds__(1024)
mx4_divide_plan_kernel(const int* __restrict__ plan, int experts, int limit, int few_tile, int max_few, int max_many, int* __restrict__ few,
                       int* __restrict__ many, int* error_word) {
  __shared__ int before[2][32];
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  const int first = plan[1 + min(e, experts)], slots = e < experts ? plan[1 + e + 1] - first : 0;
  const int tiles[2] = {slots <= limit ? (slots + few_tile - 1) / few_tile : 0, slots > limit ? (slots + MXP_TILE - 1) / MXP_TILE : 0};
  int run[2] = {tiles[0], tiles[1]};
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, run[kind], offset);
      if (lane >= offset) run[kind] += other;
    }
    if (lane == 31) before[kind][warp] = run[kind];
  }
  __syncthreads();
  int* plans[2] = {few, many};
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const int size = kind ? MXP_TILE : few_tile, most = kind ? max_many : max_few;
    int at = run[kind] - tiles[kind], all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += before[kind][w];
      all += before[kind][w];
    }
    if (e == 0) {
      plans[kind][0] = min(all, most);
      if (all > most) atomicOr(error_word, SRB_FLAG_BAD_SLOT);
    }
    if (e < experts) plans[kind][1 + e] = first;
    if (e == experts - 1) plans[kind][1 + experts] = first + slots;
    int* list = plans[kind] + 1 + experts + 1;
    for (int t = 0; t < tiles[kind]; ++t)
      if (at + t < most) {
        list[2 * (at + t)] = e;
        list[2 * (at + t) + 1] = first + t * size;
      }
  }
}
extern "C" int srb_mx4_divide_plan(const int* plan, int experts, int limit, int few_tile, int max_few, int max_many, int* few, int* many, int* error_word,
                                   void* stream) {
  if (experts <= 0 || experts > 1024) SRB_FAIL("mx4_divide_plan: %d experts are outside 1 .. 1024", experts);
  if (limit < 0 || few_tile <= 0) SRB_FAIL("mx4_divide_plan: experts of up to %d slots in tiles of %d", limit, few_tile);
  SRB_CUDA_CALL(srb_launch(mx4_divide_plan_kernel, dim3(1), dim3(1024), 0, (cudaStream_t)stream, plan, experts, limit, few_tile, max_few, max_many, few, many,
                           error_word));
  return SRB_OK;
}
