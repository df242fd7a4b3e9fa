// Rows of 4-bit floating point values with scales at two levels:
//     value[r][c] = code[r][c] * block[r][c / 16] * scale[r],
// codes e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), block scales e4m3 (up to 448), row scales float32:
//     inv = 2688 / max|x_r|  (2688 = 6 * 448),  scale = max|x_r| * fl(1/2688),
//     block = e4m3(max|x_b| * inv * fl(1/6)),   code = e2m1(x * (inv / block)),
// every step rounded to nearest in float32.  A row whose largest magnitude is below 2^-100 (inv / block might overflow) is
// held as zeros with scale 0; a row that holds an infinity or a NaN gets the scale NaN.
//
// Codes lie two to a byte, the even column in the low half, in rows of `pitch` bytes (16-byte aligned).  The block scales lie
// as the tensor core takes them: for 128 rows and 256 columns 2048 bytes together (in the order of row blocks, then column
// blocks), in them 512 bytes for 64 columns, and in those the four scales of row r at byte (r % 32) * 16 + (r / 32) * 4.
// Rows and columns behind the ends are zeros there.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "row_reader.cuh"

namespace tthrml {
namespace {

__host__ __device__ constexpr int64_t fp4_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// Bytes of the block scales of a matrix, and the place of those of row r for the 64 columns from c on.
__host__ __device__ constexpr int64_t fp4_scale_bytes(int64_t rows, int64_t cols) {
  return fp4_up(rows, 128) / 128 * (fp4_up(cols, 256) / 256) * 2048;
}
__device__ __forceinline__ int64_t fp4_scale_at(int64_t r, int64_t c, int64_t k_blocks) {
  return ((r >> 7) * k_blocks + (c >> 8)) * 2048 + ((c >> 6) & 3) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

struct Fp4RowScale {
  float inv;    // 2688 / max|x|, or 0
  float scale;  // max|x| / 2688, 0 or NaN
};
__device__ __forceinline__ Fp4RowScale fp4_row_scale(uint32_t top_bits) {
  Fp4RowScale r;
  if (top_bits >= 0x7F800000u) {
    r.inv = 0.0f;
    r.scale = __uint_as_float(0x7FC00000u);
  } else if (top_bits < 0x0D800000u) {  // 2^-100
    r.inv = 0.0f;
    r.scale = 0.0f;
  } else {
    const float top = __uint_as_float(top_bits);
    r.inv = __fdiv_rn(2688.0f, top);
    r.scale = __fmul_rn(top, 1.0f / 2688.0f);
  }
  return r;
}
__device__ __forceinline__ float fp4_block_value(uint32_t e4m3) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)e4m3, __NV_E4M3)));
}
// The scale of a block whose largest magnitude is `most`.
__device__ __forceinline__ uint32_t fp4_block_scale(float most, float inv) {
  return __nv_cvt_float_to_fp8(__fmul_rn(__fmul_rn(most, inv), 1.0f / 6.0f), __NV_SATFINITE, __NV_E4M3);
}
// inv / block for any block scale from the eight quotients of inv by 1, 9/8, ..., 15/8, which the lanes of a warp hold (lane j
// that by 1 + (j % 8) / 8): e4m3 is such a number times a power of two, by which a quotient scales exactly.
__device__ __forceinline__ float fp4_quotients(float inv) {
  return __fdiv_rn(inv, 1.0f + 0.125f * (float)(threadIdx.x & 7));
}
__device__ __forceinline__ float fp4_code_factor(uint32_t block, float quotients) {
  const uint32_t bits = __float_as_uint(fp4_block_value(block));
  const float q = __shfl_sync(0xffffffffu, quotients, (int)(bits >> 20) & 7);
  return block ? __fmul_rn(q, __uint_as_float((254u << 23) - (bits & 0x7F800000u))) : 0.0f;
}
// Eight codes in a word.
__device__ __forceinline__ uint32_t fp4_codes8(const float (&f)[8], float factor) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(f[i], factor);
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return w;
}

}  // namespace
}  // namespace tthrml
