// What the kernels of the 4-bit products share: the block-scaled MMA, the scales' way into tensor memory, tensor maps.
#pragma once

#include "fp4_common.cuh"
#include "tc_common.cuh"

namespace tthrml {
namespace {

constexpr int kScales = 2048;  // bytes of the block scales of 128 rows and 256 columns

// Instruction descriptor: D float32, A and B e2m1, K-major, scales e4m3 (one per 16 columns).
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                         uint32_t b_scales, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate));
}
// 32 rows of 16 bytes that lie one behind the other: groups of eight rows 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t scales_desc(const void* p) {
  const uint64_t addr = (uint64_t)(smem_u32(p) >> 4) & 0x3FFFull;
  return addr | (1ull << 16) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc));
}

// Tensor map of a byte matrix [rows][cols] with rows `pitch` bytes apart, in (box_rows x 128) tiles, 128-byte swizzle.
inline int make_map_codes(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, uint32_t box_rows) {
  EncodeTiledFn fn;
  int rc = encode_fn(&fn);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128u, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for %lld x %lld bytes of codes", (int)r, (long long)rows, (long long)cols);
    return TTHRML_ERR_CUDA;
  }
  return TTHRML_OK;
}
// The block scales as rows of 1024 bytes, read two at a time: those of 128 rows and 256 columns.
inline int make_map_scales(CUtensorMap* map, const void* base, int64_t rows, int64_t cols) {
  EncodeTiledFn fn;
  int rc = encode_fn(&fn);
  if (rc) return rc;
  const cuuint64_t dims[2] = {256, (cuuint64_t)(fp4_scale_bytes(rows, cols) / 1024)};
  const cuuint64_t strides[1] = {1024};
  const cuuint32_t box[2] = {256u, 2u};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for the scales of %lld x %lld values", (int)r, (long long)rows, (long long)cols);
    return TTHRML_ERR_CUDA;
  }
  return TTHRML_OK;
}

}  // namespace
}  // namespace tthrml
