// Rows of float elements in 16-byte vectors, from any address and stride, and the largest magnitude of such vectors.
#pragma once

#include "int8_common.cuh"

namespace tthrml {
namespace {

// How the 16-byte vectors of a row are read: at aligned addresses, as two aligned vectors shifted together, or by elements.
enum : int { kElements = 0, kAligned = 1, kShifted = 2 };

// 16 bytes from any address whose aligned surroundings hold bytes of the row on both sides.
__device__ __forceinline__ uint4 load_shifted(const char* p, uint32_t off) {
  const uint4* q = reinterpret_cast<const uint4*>(p - off);
  const uint4 a = __ldg(q), b = __ldg(q + 1);
  uint32_t w[5];
  const uint32_t word = off >> 2, bits = (off & 3u) * 8u;  // the same for the whole row
  if (word == 0)
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x;
  else if (word == 1)
    w[0] = a.y, w[1] = a.z, w[2] = a.w, w[3] = b.x, w[4] = b.y;
  else if (word == 2)
    w[0] = a.z, w[1] = a.w, w[2] = b.x, w[3] = b.y, w[4] = b.z;
  else
    w[0] = a.w, w[1] = b.x, w[2] = b.y, w[3] = b.z, w[4] = b.w;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}

template <typename T, bool ALIGNED>
struct RowReader {
  const T* x;
  int32_t cols;
  int64_t cs;
  int mode;
  uint32_t off;
  __device__ __forceinline__ Vec8<T> vector(int32_t c) const {  // elements c .. c + 7, zeros behind the end
    Vec8<T> v;
    if ((ALIGNED || mode != kElements) && c + 8 <= cols) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        v.w[i] = ALIGNED || mode == kAligned ? __ldg(reinterpret_cast<const uint4*>(x + c) + i)
                                             : load_shifted(reinterpret_cast<const char*>(x + c) + 16 * i, off);
      return v;
    }
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) v.w[i] = make_uint4(0u, 0u, 0u, 0u);
    if (c < cols) {
      T* e = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < cols) e[i] = x[(int64_t)(c + i) * cs];
    }
    return v;
  }
};

// Running maximum of magnitudes, NaN once one is met: 16-bit elements two at a time.
struct MaxF32 {
  float top = 0.0f;
  __device__ __forceinline__ void add(const uint4& v) {
    top = max_abs(max_abs(max_abs(max_abs(top, __uint_as_float(v.x)), __uint_as_float(v.y)), __uint_as_float(v.z)),
                  __uint_as_float(v.w));
  }
  __device__ __forceinline__ float value() const { return top; }
};
template <typename T2>
struct MaxPacked {
  uint32_t top = 0u;
  __device__ __forceinline__ void add(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = w[i] & 0x7FFF7FFFu;
      const T2 t = __hmax2_nan(*reinterpret_cast<const T2*>(&top), *reinterpret_cast<const T2*>(&m));
      top = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  __device__ __forceinline__ float value() const {
    const T2 t = *reinterpret_cast<const T2*>(&top);
    return max_abs(to_f32(t.x), to_f32(t.y));
  }
};
template <typename T>
struct MaxOf;
template <>
struct MaxOf<float> : MaxF32 {};
template <>
struct MaxOf<__nv_bfloat16> : MaxPacked<__nv_bfloat162> {};
template <>
struct MaxOf<__half> : MaxPacked<__half2> {};

template <typename T>
__device__ __forceinline__ void add_vector(MaxOf<T>& most, const Vec8<T>& v) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) most.add(v.w[i]);
}

}  // namespace
}  // namespace tthrml
