// Element types of the operators' inputs and outputs, and the quantisation of a row to 8-bit integers:
//     scale = max|x| * fl(1/127),   q = rint(x * fl(127 / max|x|)).
// A row whose largest magnitude is below 2^-120 (127 / max|x| would overflow) is held as zeros with scale 0; a
// row that holds an infinity or a NaN gets the scale NaN, so every value computed from it is NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tthrml {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements from a 16-byte aligned address.
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) v.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T>& v, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
}

// Magnitude as an integer that orders like the float (NaN above infinity), for maxima that must not lose a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

struct RowScale {
  float inv;    // 127 / max|x|, or 0
  float scale;  // max|x| / 127, 0 or NaN
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
  RowScale r;
  if (top_bits >= 0x7F800000u) {
    r.inv = 0.0f;
    r.scale = __uint_as_float(0x7FC00000u);
  } else if (top_bits < 0x03800000u) {  // 2^-120
    r.inv = 0.0f;
    r.scale = 0.0f;
  } else {
    const float top = __uint_as_float(top_bits);
    r.inv = __fdiv_rn(127.0f, top);
    r.scale = __fmul_rn(top, 0.007874015718698502f);  // fl(1/127)
  }
  return r;
}
// rint(x inv) in the low byte of a word: |x| <= max|x| makes |x inv| at most 127 (1 + 2^-23), so no clamp is needed, and 3 2^22
// added rounds to the nearest integer, ties to even.  (A row that is not finite has inv = 0 and may get any byte: its
// scale is NaN.)
__device__ __forceinline__ uint32_t quantize_low(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float inv) {
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = quantize_low(f[i], inv);
  return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}
// The larger of a maximum and the magnitude of v, NaN if either is.
__device__ __forceinline__ float max_abs(float top, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(v)));
  return r;
}

inline int64_t dtype_bytes(int32_t dtype) {
  switch (dtype) {
    case TTHRML_DT_F32: return 4;
    case TTHRML_DT_BF16:
    case TTHRML_DT_F16: return 2;
    case TTHRML_DT_I8: return 1;
    default: return 0;
  }
}

}  // namespace
}  // namespace tthrml
