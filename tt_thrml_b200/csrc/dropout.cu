// Dropout by a counter-based generator; the mask is never stored, the backward pass draws it again:
//     y[i] = keep[i] ? x[i] * 65536 / (65536 - cut) : 0,   keep[i] = (half-word i % 8 of draw i / 8) >= cut,
// draw g = Philox4x32-10 keyed by the seed at counter (g, g >> 32, step, "DROP"), half-words from the low half of its first
// word on.  A 16-bit half decides an element: the probability is cut / 65536 exactly, and so is the factor that keeps the mean,
// and one draw serves eight elements (a 32-bit word each would double the instructions to 18 per element).  Dropped elements
// are 0 whatever they held.
//
// Bound: memory (an element read and written).  A draw is 40 instructions with 64-bit products and the round keys at hand, 5
// per element, about as many as the scaling and the choice; four groups per thread hide them behind the loads.  67 M
// bfloat16: 46 us (5.8 TB/s); with 32-bit products, keys added up and masks built per half-word 67 us.  67 M float32: 80 us.
#include "int8_common.cuh"

namespace tthrml {
namespace {

constexpr uint32_t kSaltDropout = 0x44524F50u;  // "DROP"
constexpr int kGroups = 4;                      // of eight elements per thread, a block's width apart

struct DropoutArgs {
  const void* x;
  void* y;
  int64_t n;
  uint32_t cut;
  float scale;
  uint64_t seed;
  uint32_t step;
  const void* step_at;  // the step on the device, or NULL
  int32_t step_wide;
  uint32_t* step_used;  // where it is left for the backward pass, or NULL
};

// Philox4x32-10 with 64-bit products and the round keys at hand: four instructions a round.
__device__ __forceinline__ u32x4 draw8(int64_t g, uint32_t step, const PhiloxKeys& k) {
  u32x4 c = {(uint32_t)g, (uint32_t)(g >> 32), step, kSaltDropout};
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
    c = u32x4{(uint32_t)(p1 >> 32) ^ c.y ^ k.a[r], (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.b[r], (uint32_t)p0};
  }
  return c;
}
template <typename T>
__device__ __forceinline__ uint32_t packed_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t packed_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t packed_pair<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ Vec8<T> dropped(const Vec8<T>& v, const u32x4& draw, uint32_t cut16, bool all, float scale) {
  float f[8];
  unpack8(v, f);
  Vec8<T> o;
  uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t bits = word_of(draw, q);  // a half against the cut: shifted to the top, whole words
    const float lo = (bits << 16) >= cut16 && !all ? __fmul_rn(f[2 * q], scale) : 0.0f;
    const float hi = bits >= cut16 && !all ? __fmul_rn(f[2 * q + 1], scale) : 0.0f;
    if constexpr (sizeof(T) == 4) {
      w[2 * q] = __float_as_uint(lo);
      w[2 * q + 1] = __float_as_uint(hi);
    } else {
      w[q] = packed_pair<T>(lo, hi);
    }
  }
  return o;
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) k_dropout(const DropoutArgs a) {
  uint32_t step = a.step;
  if (a.step_at)
    step = a.step_wide ? (uint32_t)__ldg(reinterpret_cast<const unsigned long long*>(a.step_at))
                       : (uint32_t)__ldg(reinterpret_cast<const unsigned int*>(a.step_at));
  if (a.step_used && blockIdx.x == 0 && threadIdx.x == 0) *a.step_used = step;
  const PhiloxKeys keys = philox_keys(seed_lo(a.seed), seed_hi(a.seed));
  const uint32_t cut16 = a.cut << 16;  // a cut of 65536 leaves nothing
  const bool all = a.cut == 65536u;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  const int64_t groups = (a.n + 7) / 8;
  for (int64_t first = (int64_t)blockIdx.x * (256 * kGroups) + threadIdx.x; first < groups;
       first += (int64_t)gridDim.x * (256 * kGroups)) {
    Vec8<T> v[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int64_t at = (first + 256 * j) * 8;
      if (ALIGNED && at + 8 <= a.n) {
        v[j] = load8(x + at);
      } else {
        T* e = reinterpret_cast<T*>(&v[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = at + i < a.n ? x[at + i] : from_f32<T>(0.0f);
      }
    }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int64_t g = first + 256 * j, at = g * 8;
      if (at >= a.n) break;
      const Vec8<T> o = dropped(v[j], draw8(g, step, keys), cut16, all, a.scale);
      if (ALIGNED && at + 8 <= a.n) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(y + at)[i] = o.w[i];
      } else {
        const T* e = reinterpret_cast<const T*>(&o);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (at + i < a.n) y[at + i] = e[i];
      }
    }
  }
}

template <typename T>
int launch(const DropoutArgs& a, cudaStream_t st) {
  const int64_t blocks = ((a.n + 7) / 8 + 256 * kGroups - 1) / (256 * kGroups);
  const unsigned grid = (unsigned)(blocks < 148 * 64 ? blocks : 148 * 64);
  if ((uintptr_t)a.x % 16 == 0 && (uintptr_t)a.y % 16 == 0)
    k_dropout<T, true><<<grid, 256, 0, st>>>(a);
  else
    k_dropout<T, false><<<grid, 256, 0, st>>>(a);
  return launch_status("k_dropout launch");
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_dropout(const void* x, int32_t dtype, int64_t n, int32_t cut, uint64_t seed, uint32_t step,
                              const void* step_at, int32_t step_wide, uint32_t* step_used, void* y, void* stream) {
  using namespace tthrml;
  if (n == 0) return TTHRML_OK;
  if (!x || !y) {
    set_error("tthrml_dropout: NULL argument");
    return TTHRML_ERR_ARG;
  }
  const int64_t bytes = dtype_bytes(dtype);
  if (dtype == TTHRML_DT_I8 || bytes == 0) {
    set_error("tthrml_dropout: elements must be float32, bfloat16 or float16 (got code %d)", (int)dtype);
    return TTHRML_ERR_ARG;
  }
  if (n < 0 || n > (int64_t)1 << 56 || cut < 0 || cut > 65536 || (uintptr_t)x % bytes || (uintptr_t)y % bytes ||
      (step_at && (uintptr_t)step_at % (step_wide ? 8 : 4))) {
    set_error("tthrml_dropout: elements, cut or alignment out of range (%lld elements, cut %d of 0 to 65536)", (long long)n,
              (int)cut);
    return TTHRML_ERR_ARG;
  }
  const DropoutArgs a = {x, y, n, (uint32_t)cut, cut == 65536 ? 0.0f : (float)(65536.0 / (65536.0 - cut)), seed, step, step_at,
                         step_wide, step_used};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TTHRML_DT_F32) return launch<float>(a, st);
  if (dtype == TTHRML_DT_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<__half>(a, st);
}
