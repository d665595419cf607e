// The block-scaled tensor-core instructions of sm_100 (tcgen05.mma ... block_scale) and what feeds them.
//
// Operands lie in shared memory in rows of 128 bytes with the 128-byte swizzle, as for the plain products; a step takes 32 bytes of a row: 64
// four-bit entries (kind mxf4), or 32 entries of eight bits (kind mxf8f6f4), where four-bit entries stand 16 to 16 bytes, eight bytes of
// codes and eight that are not read.  Scales lie in tensor memory: row r's in lane r % 32 (of every quarter of the lanes) and
// column r / 32, a byte for each of four consecutive blocks of 32 entries; the instruction descriptor says which bytes a step takes, and the
// address may be an even column alone (an odd one faults).
#pragma once
#include "common.cuh"
#include "tcgen05_helpers.cuh"
#include <atomic>
#include <mutex>

#define MX_E4M3 0u
#define MX_E2M1 5u       // among the types of kind mxf8f6f4

// kind mxf8f6f4: scales of 2^n, both operands K-major, M = 128.  The scale byte `k` of a word is ORed in by mx_idesc_step.
__device__ __forceinline__ unsigned mx_idesc(unsigned a_type, unsigned b_type, int m, int n) {
  return (a_type << 7) | (b_type << 10) | ((unsigned)(n >> 3) << 17) | (1u << 23) | ((unsigned)(m >> 4) << 24);
}
__device__ __forceinline__ unsigned mx_idesc_step(unsigned idesc, unsigned byte) { return idesc | (byte << 4) | (byte << 29); }

// kind mxf4: both operands in four bits, packed
__device__ __forceinline__ unsigned mx_idesc_four(int m, int n) { return (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | (1u << 23) | ((unsigned)(m >> 4) << 24); }
__device__ __forceinline__ void umma_mx4(unsigned tmem_d, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned a_scales,
                                         unsigned b_scales, unsigned accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate) : "memory");
}
// 512 bytes of shared memory, 32 rows of 16, to four columns of all lanes (every quarter gets the 32 rows)
__device__ __forceinline__ void tmem_copy_scales(unsigned tmem, unsigned long long desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// rows of 16 bytes without swizzle, groups of eight rows 128 bytes apart
__device__ __forceinline__ unsigned long long scales_descriptor(unsigned address) {
  return (unsigned long long)((address & 0x3ffffu) >> 4) | ((unsigned long long)(128u >> 4) << 32) | (1ull << 46);
}

// Lets the kernel have that much shared memory, once for a device and a size (`allowed`: what a device was told last).
#define MX4_MAX_DEVICES 64
static inline int mx4_allow_shared(const void* kernel, int bytes, std::atomic<int>* allowed) {
  int device = 0;
  SRB_CUDA_CALL(cudaGetDevice(&device));
  if (device < MX4_MAX_DEVICES && allowed[device].load() >= bytes) return SRB_OK;
  SRB_CUDA_CALL(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (device < MX4_MAX_DEVICES) {
    int told = allowed[device].load();
    while (told < bytes && !allowed[device].compare_exchange_weak(told, bytes)) {}
  }
  return SRB_OK;
}

// ---- maps for TMA ----------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &result) == cudaSuccess &&
        result == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(entry);
  });
  return fn;
}

// A matrix [rows, columns] of elements of `type`, `pitch` bytes apart, cut into boxes.
static inline int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, long long columns, long long pitch,
                    int box_rows, int box_columns, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) SRB_FAIL("four-bit products: the driver does not offer cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows};
  const cuuint32_t element[2] = {1, 1};
  const CUresult status = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, element, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (status != CUDA_SUCCESS) SRB_FAIL("four-bit products: cuTensorMapEncodeTiled failed with %d", (int)status);
  return SRB_OK;
}
static inline int make_bytes_map(CUtensorMap* map, const void* base, long long rows, long long bytes, int box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, bytes, bytes, box_rows, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Codes that stand 16 to 16 bytes in shared memory, as kind mxf8f6f4 takes them (a box of 128 entries is 128 bytes a row there; the barrier
// counts the 64 bytes of codes).  Base on a 32-byte border, `k_tiles` * 64 bytes a row.
static inline int make_codes_map(CUtensorMap* map, const void* base, long long rows, int k_tiles, int box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, base, rows, k_tiles * 128ll, k_tiles * 64ll, box_rows, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}
static inline int make_scales_map(CUtensorMap* map, const void* base, long long tiles, int at_once) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, tiles, 128, 512, at_once, 128, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// ---- pairs of CTAs (cta_group::2): M = 256, the even CTA's thread issues for both -----------------------------------------
__device__ __forceinline__ void umma_mx4_pair(unsigned tmem_d, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned a_scales,
                                              unsigned b_scales, unsigned accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_mx8_pair(unsigned tmem_d, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned a_scales,
                                              unsigned b_scales, unsigned accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate) : "memory");
}
// in both CTAs, each from its own shared memory
__device__ __forceinline__ void tmem_copy_scales_pair(unsigned tmem, unsigned long long desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// A bounded wait on a barrier on which the other CTA's threads arrive too.
__device__ __forceinline__ bool mbar_wait_warp_cluster(unsigned bar, unsigned parity, volatile int* abort_flag) {
  const long long start = clock64();
  bool done = false;
  for (unsigned spins = 0; !done; ++spins) {
    unsigned ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    done = ok != 0;
    if (!done && (spins & 255u) == 255u) {
      if (*abort_flag) break;
      if (clock64() - start > SRB_SPIN_LIMIT) {
        *abort_flag = 1;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, done);
}
