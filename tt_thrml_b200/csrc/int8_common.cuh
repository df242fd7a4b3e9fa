// Element types of the operators' inputs and outputs, and the quantisation of a row to 8-bit integers:
//     scale = max|x| * fl(1/127),   q = rint(x * fl(127 / max|x|)) clamped to +-127.
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
// NaN times inv = 0 stays NaN; its conversion gives 0.
__device__ __forceinline__ int32_t quantize(float x, float inv) {
  const int32_t q = __float2int_rn(__fmul_rn(x, inv));
  return max(-127, min(127, q));
}
__device__ __forceinline__ uint32_t pack4(int32_t a, int32_t b, int32_t c, int32_t d) {
  return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
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
