// AdamW (Adam with decoupled weight decay; Loshchilov and Hutter, ICLR 2019) over many tensors in one launch:
//     m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//     p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with the moments in float32 or in 8-bit codes.  All arithmetic is float32; the moments round after every operation.
//
// Bound: memory.  Each element of the tensors and moments is read once and written once: 2 p + g + 16 bytes with
// float32 moments, 2 p + g + 4 + 1/16 with codes (p, g: bytes of a parameter and a gradient).
//
// The tensors' addresses travel in the launch's parameters, so a step uploads nothing and a captured graph keeps its
// own copy.  The moments of all tensors lie in one buffer, each tensor's segment padded to 256 elements.  The CTAs walk
// side by side over 2048-element chunks of the concatenated tensors (a chunk never spans two tensors); a warp holds 256
// of them, a thread two groups of four 128 apart, so that every load and store of a warp is contiguous.  33.6 M float32
// weights take 142 us so (6.6 TB/s, the measured copy rate); of 154 us, a range of chunks of its own for each CTA made 167,
// eight adjacent elements per thread 178.  With codes 138 us (instruction issue).
//
// The step counter and the learning rate stand in device memory, so a replayed graph counts on; in a step's last launch the
// last CTA that has read the counter advances it.
//
// 8-bit codes, one warp per block of 256 elements with the block's largest |m| and v as scales:
//     m = sign q^2 max|m| / 127^2, q = 0..127;      v = q^4 max v / 255^4, q = 0..255.
// The powers give small values small steps: v spans 255^4 = 2^32, that is 2^16 in gradient magnitude.  A value is
// rounded to the code below or above at random with the probability that keeps its mean, because a code's step exceeds
// what one step of the averages changes ((1 - b2) = 0.1 % of v): rounding to nearest would hold them where they are.
// The random words are Philox4x32-10 at (element / 4, element / 4 >> 32, step, "ADMW"), word element % 4, low half
// for m and high half for v, so a run can be repeated.  A v > 0 is never rounded to zero, or m / (0 + eps) would
// follow.  A block whose largest v is below 2^-90 is held as zeros; one that takes in an infinity or a NaN is NaN.
#include <cmath>
#include <type_traits>

#include "int8_common.cuh"

namespace tthrml {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kChunk = 8 * kAdamThreads;
constexpr uint32_t kSaltAdam = 0x41444D57u;  // "ADMW"

template <int T>
struct AdamTable {
  tthrml_adamw_tensor t[T];
  int32_t first_chunk[T + 1];
};

struct AdamArgs {
  void* m;          // float32 or int8 [elements]
  void* v;          // float32 or uint8 [elements]
  float* m_scale;   // [elements / 256], codes only
  float* v_scale;
  tthrml_adamw_ctl* ctl;
  float b1, d1, b2, d2, eps;  // d = 1 - b
  float minus_zero;
  double beta1, beta2, weight_decay;
  uint64_t seed;
  int32_t n_tensors;
  int32_t last;     // this launch ends the step
};

// The bits of four consecutive elements from place i of a tensor of n (16-bit elements in the first two words);
// `vectors`: the tensor is aligned to four elements.  Loading and converting are apart, so that a thread's loads are all on
// their way before the first conversion waits for one.
struct Raw4 {
  uint32_t w[4];
};
__device__ __forceinline__ Raw4 load_raw(int32_t dtype, const void* base, int64_t i, int64_t n, bool vectors) {
  Raw4 r = {{0u, 0u, 0u, 0u}};
  if (dtype == TTHRML_DT_F32) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(base) + i;
    if (vectors && i + 4 <= n) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) r.w[k] = p[k];
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + i;
    if (vectors && i + 4 <= n) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      r.w[0] = v.x, r.w[1] = v.y;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) r.w[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
    }
  }
  return r;
}
__device__ __forceinline__ void convert(int32_t dtype, const Raw4& r, float2 (&f)[2]) {
  if (dtype == TTHRML_DT_F32) {
    f[0] = make_float2(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]));
    f[1] = make_float2(__uint_as_float(r.w[2]), __uint_as_float(r.w[3]));
  } else if (dtype == TTHRML_DT_BF16) {
#pragma unroll
    for (int k = 0; k < 2; ++k) f[k] = make_float2(__uint_as_float(r.w[k] << 16), __uint_as_float(r.w[k] & 0xFFFF0000u));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) f[k] = __half22float2(*reinterpret_cast<const __half2*>(&r.w[k]));
  }
}
template <typename T>
__device__ __forceinline__ void store_elems(void* base, int64_t i, int64_t n, bool vectors, const float2 (&f)[2]) {
  T* p = reinterpret_cast<T*>(base) + i;
  if (vectors && i + 4 <= n) {
    if (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    } else {
      uint2 v;
      T* e = reinterpret_cast<T*>(&v);
      e[0] = from_f32<T>(f[0].x), e[1] = from_f32<T>(f[0].y), e[2] = from_f32<T>(f[1].x), e[3] = from_f32<T>(f[1].y);
      *reinterpret_cast<uint2*>(p) = v;
    }
  } else {
    if (i < n) p[0] = from_f32<T>(f[0].x);
    if (i + 1 < n) p[1] = from_f32<T>(f[0].y);
    if (i + 2 < n) p[2] = from_f32<T>(f[1].x);
    if (i + 3 < n) p[3] = from_f32<T>(f[1].y);
  }
}
__device__ __forceinline__ void store_any(int32_t dtype, void* base, int64_t i, int64_t n, bool vectors, const float2 (&f)[2]) {
  if (dtype == TTHRML_DT_F32)
    store_elems<float>(base, i, n, vectors, f);
  else if (dtype == TTHRML_DT_BF16)
    store_elems<__nv_bfloat16>(base, i, n, vectors, f);
  else
    store_elems<__half>(base, i, n, vectors, f);
}

// Pairs of elements: one packed instruction for two float32 operations, each rounded as the single one.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
// A product that goes into a sum: packed products and sums are contracted to one rounding, even with their rounding named,
// and codes and scales have to be those of the formula bit for bit.  -0, which leaves the product as it is, comes as a
// value that the compiler does not know.
__device__ __forceinline__ float2 product2(float2 a, float2 b, float minus_zero) { return __ffma2_rn(a, b, both(minus_zero)); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

// Byte j of a word under the exponent of 2^23: 2^23 + byte.
__device__ __forceinline__ float byte_high(uint32_t w, int j) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540u | (uint32_t)j));
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The same with subnormal arguments, which the other one takes for 0.
__device__ __forceinline__ float sqrt_subnormal(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// floors of 0 <= x < 2^22
__device__ __forceinline__ float2 floor2(float2 x) { return add2(__fadd2_rd(x, both(8388608.0f)), both(-8388608.0f)); }
// h + 1/2 of the low (high) half words h: 65536 times a uniform that is never 0 or 1
__device__ __forceinline__ float2 low_halves(uint32_t a, uint32_t b) {
  return add2(make_float2(__uint_as_float(__byte_perm(a, 0x4B000000u, 0x7410u)),
                          __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7410u))),
              both(-8388607.5f));
}
__device__ __forceinline__ float2 high_halves(uint32_t a, uint32_t b) {
  return add2(make_float2(__uint_as_float(__byte_perm(a, 0x4B000000u, 0x7432u)),
                          __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7432u))),
              both(-8388607.5f));
}
__device__ __forceinline__ float fourth(float k) {
  const float k2 = __fmul_rn(k, k);
  return __fmul_rn(k2, k2);
}
__device__ __forceinline__ float2 fourth2(float2 k, float minus_zero) {  // k^2 is exact, k^4 rounds
  const float2 k2 = mul2(k, k);
  return product2(k2, k2, minus_zero);
}

// The approximate roots are off by one only next to a whole number: the place of y among the squares (fourth powers) again.
__device__ __noinline__ float2 place_m(float y, float k) {  // (k, y - k^2)
  if (__fmul_rn(k, k) > y) k -= 1.0f;
  if (__fmul_rn(k + 1.0f, k + 1.0f) <= y) k += 1.0f;
  return make_float2(k, __fsub_rn(y, __fmul_rn(k, k)));
}
__device__ __noinline__ float2 place_v(float y, float k) {  // (k, y - k^4)
  if (fourth(k) > y) k -= 1.0f;
  if (fourth(k + 1.0f) <= y) k += 1.0f;
  return make_float2(k, __fsub_rn(y, fourth(k)));
}

// Whether a remainder lies outside [0, span): a negative one is the larger unsigned integer.
__device__ __forceinline__ bool outside(float over, float span) { return __float_as_uint(over) >= __float_as_uint(span); }

// Codes of y = |m| 127^2 / max|m|: the largest k with k^2 <= y, or k + 1 with probability (y - k^2) / (2 k + 1).  u65536 is
// 65536 times the uniform; the scaling by powers of two is exact.
__device__ __forceinline__ float2 codes_m(float2 y, float2 u65536) {
  float2 k = floor2(make_float2(sqrt_approx(y.x), sqrt_approx(y.y)));
  float2 over = __ffma2_rn(neg2(k), k, y), span = __ffma2_rn(k, both(2.0f), both(1.0f));  // k^2 and 2 k + 1 are exact
  if (outside(over.x, span.x) || outside(over.y, span.y)) {
    const float2 a = place_m(y.x, k.x), b = place_m(y.y, k.y);
    k = make_float2(a.x, b.x);
    over = make_float2(a.y, b.y);
    span = __ffma2_rn(k, both(2.0f), both(1.0f));
  }
  const float2 t = mul2(u65536, span), o = mul2(over, both(65536.0f)), n = add2(k, both(1.0f));
  return make_float2(fminf(t.x < o.x ? n.x : k.x, 127.0f), fminf(t.y < o.y ? n.y : k.y, 127.0f));
}
// Codes of y = v 255^4 / max v, likewise with fourth powers; a y > 0 gets at least 1.
__device__ __forceinline__ float2 codes_v(float2 y, float2 u65536, float minus_zero) {
  float2 k = floor2(make_float2(sqrt_approx(sqrt_approx(y.x)), sqrt_approx(sqrt_approx(y.y))));
  float2 n = add2(k, both(1.0f)), k4 = fourth2(k, minus_zero), n4 = fourth2(n, minus_zero), over = add2(y, neg2(k4));
  float2 span = add2(n4, neg2(k4));
  if (outside(over.x, span.x) || outside(over.y, span.y)) {
    const float2 a = place_v(y.x, k.x), b = place_v(y.y, k.y);
    k = make_float2(a.x, b.x);
    over = make_float2(a.y, b.y);
    n = add2(k, both(1.0f));
    span = add2(fourth2(n, minus_zero), neg2(fourth2(k, minus_zero)));
  }
  // k = 0 takes no chances: 1 wherever y > 0
  const float2 t = mul2(mul2(u65536, span), make_float2(fminf(k.x, 1.0f), fminf(k.y, 1.0f))), o = mul2(over, both(65536.0f));
  return make_float2(fminf(t.x < o.x ? n.x : k.x, 255.0f), fminf(t.y < o.y ? n.y : k.y, 255.0f));
}
// b^t by squaring, t >= 1: the library's power is a few hundred instructions on the way of a small step's only round.  At most
// 2 log2 t roundings of 2^-53, and none at t = 1, where 1 - b is smallest.
__device__ __forceinline__ double power(double b, int64_t t) {
  double r = 1.0;
  for (;; b *= b) {
    if (t & 1) r *= b;
    t >>= 1;
    if (t == 0) return r;
  }
}

// The tensor that holds chunk c: the last of n whose first chunk is not behind c.  A warp looks at 32 places at a time.
__device__ __forceinline__ int tensor_of(const int32_t* first_chunk, int n, int c) {
  const int lane = threadIdx.x & 31, stride = (n + 31) / 32;
  int at = lane * stride;
  const int found = 31 - __clz(__ballot_sync(0xffffffffu, at < n && first_chunk[at] <= c));
  if (stride == 1) return found;
  at = found * stride + lane;  // stride <= 32
  return found * stride + 31 - __clz(__ballot_sync(0xffffffffu, at < n && first_chunk[at] <= c));
}

// ROOTS (codes): subnormal v have roots of their own (flushes_roots).
template <int BITS, int T, bool ROOTS>
__global__ void __launch_bounds__(kAdamThreads, 4)
    k_adamw(const __grid_constant__ AdamTable<T> tab, const __grid_constant__ AdamArgs a) {
  __shared__ float coef[4];  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd, step
  static_assert(T <= 1024, "two rounds of 32 places");
  const int chunks = tab.first_chunk[a.n_tensors];
  // The table by generic addresses: its lookups are by a warp's lanes, and a constant bank serves one address at a time.
  const AdamTable<T>* table = &tab;
  asm("" : "+l"(table));
  int ti = 0;
  const int place = 256 * (threadIdx.x >> 5) + 4 * (threadIdx.x & 31);
  const int64_t step = a.ctl->step + 1;
  // the coefficients in double, a warp each; every warp passes the barrier once, after its first loads are on their way
  if (threadIdx.x == 0) coef[0] = (float)(a.ctl->lr / (1.0 - power(a.beta1, step)));
  if (threadIdx.x == 32) coef[1] = (float)(1.0 / sqrt(1.0 - power(a.beta2, step)));
  if (threadIdx.x == 64) coef[2] = (float)(1.0 - a.ctl->lr * a.weight_decay);
  const auto barrier = [] { asm volatile("bar.sync 1, %0;" ::"n"(kAdamThreads) : "memory"); };
  bool ready = false;
  // The last CTA that has read the step advances the counter.  The count goes out early: nothing waits for it before the end.
  unsigned long long before = 0ull;
  const auto count = [&] {
    if (threadIdx.x == 0 && a.last) {
      __threadfence();
      before = atomicAdd(&a.ctl->ticket, 1ull);
    }
  };
  float step_size = 0.0f, r_bias2 = 0.0f, keep = 0.0f;
  const PhiloxKeys keys = philox_keys((uint32_t)a.seed, (uint32_t)(a.seed >> 32));
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    if (tab.first_chunk[ti + 1] <= c) ti = tensor_of(table->first_chunk, a.n_tensors, c);
    const tthrml_adamw_tensor& t = table->t[ti];
    const int64_t i = (int64_t)(c - table->first_chunk[ti]) * kChunk + place;
    if (i - 4 * (threadIdx.x & 31) >= t.n) continue;  // whole warps
    const int64_t e = t.state + i;  // this thread's groups: e .. e + 3 and e + 128 .. e + 131
    const bool pv = (uintptr_t)t.param % (t.param_dtype == TTHRML_DT_F32 ? 16 : 8) == 0;
    const bool gv = (uintptr_t)t.grad % (t.grad_dtype == TTHRML_DT_F32 ? 16 : 8) == 0;
    float2 p[2][2], g[2][2], m[2][2], v[2][2];
    Raw4 pr[2], gr[2];
    uint32_t mc[2], vc[2];
    float um = 0.0f, uv = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      gr[h] = load_raw(t.grad_dtype, t.grad, i + 128 * h, t.n, gv);
      pr[h] = load_raw(t.param_dtype, t.param, i + 128 * h, t.n, pv);
      if (BITS == 32) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.m) + e + 128 * h);
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.v) + e + 128 * h);
        m[h][0] = make_float2(x.x, x.y), m[h][1] = make_float2(x.z, x.w);
        v[h][0] = make_float2(y.x, y.y), v[h][1] = make_float2(y.z, y.w);
      } else {
        mc[h] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const int8_t*>(a.m) + e + 128 * h) ^ 0x80808080u;
        vc[h] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(a.v) + e + 128 * h);
      }
    }
    if (BITS == 8) {
      um = __fmul_rn(a.m_scale[e >> 8], 1.0f / 16129.0f);
      uv = __fmul_rn(a.v_scale[e >> 8], 1.0f / 4228250625.0f);
    }
    if (!ready) {
      barrier();
      step_size = coef[0], r_bias2 = coef[1], keep = coef[2];
      count();
      ready = true;
    }
    float tm = 0.0f, tv = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      convert(t.grad_dtype, gr[h], g[h]);
      convert(t.param_dtype, pr[h], p[h]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (BITS == 8) {
          const float2 c8 = add2(make_float2(byte_high(mc[h], 2 * k), byte_high(mc[h], 2 * k + 1)), both(-8388736.0f));
          const float2 mag = mul2(mul2(c8, c8), both(um));
          m[h][k] = make_float2(copysignf(mag.x, c8.x), copysignf(mag.y, c8.y));
          v[h][k] = mul2(fourth2(add2(make_float2(byte_high(vc[h], 2 * k), byte_high(vc[h], 2 * k + 1)), both(-8388608.0f)), a.minus_zero),
                         both(uv));
        }
        const float2 gk = g[h][k];
        const float2 mk = m[h][k] = add2(product2(m[h][k], both(a.b1), a.minus_zero), product2(gk, both(a.d1), a.minus_zero));
        const float2 vk = v[h][k] = add2(product2(v[h][k], both(a.b2), a.minus_zero), product2(mul2(gk, gk), both(a.d2), a.minus_zero));
        float2 upd;
        if (BITS == 32) {
          const float2 denom = add2(mul2(make_float2(__fsqrt_rn(vk.x), __fsqrt_rn(vk.y)), both(r_bias2)), both(a.eps));
          upd = make_float2(__fdiv_rn(mk.x, denom.x), __fdiv_rn(mk.y, denom.y));
        } else {
          // the hardware's root and reciprocal (2^-21 of the update at most, whose moments are codes to about 1 %): the
          // step on codes is bound by its instructions
          const float2 root = ROOTS ? make_float2(sqrt_subnormal(vk.x), sqrt_subnormal(vk.y))
                                    : make_float2(sqrt_approx(vk.x), sqrt_approx(vk.y));
          const float2 denom = add2(mul2(root, both(r_bias2)), both(a.eps));
          upd = mul2(mk, make_float2(rcp_approx(denom.x), rcp_approx(denom.y)));
          tm = max_abs(max_abs(tm, mk.x), mk.y);
          tv = max_abs(max_abs(tv, vk.x), vk.y);
        }
        p[h][k] = add2(mul2(p[h][k], both(keep)), neg2(mul2(upd, both(step_size))));
      }
      store_any(t.param_dtype, t.param, i + 128 * h, t.n, pv, p[h]);
      if (BITS == 32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.m) + e + 128 * h) =
            make_float4(m[h][0].x, m[h][0].y, m[h][1].x, m[h][1].y);
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.v) + e + 128 * h) =
            make_float4(v[h][0].x, v[h][0].y, v[h][1].x, v[h][1].y);
      }
    }
    if (BITS == 8) {
      const uint32_t bm = __reduce_max_sync(0xffffffffu, abs_bits(tm)), bv = __reduce_max_sync(0xffffffffu, abs_bits(tv));
      float top_m = __uint_as_float(bm), top_v = __uint_as_float(bv);
      const bool finite = bm < 0x7F800000u && bv < 0x7F800000u;
      if (!finite) top_m = top_v = __uint_as_float(0x7FC00000u);
      if (top_v < 8.0779356694631609e-28f) top_v = 0.0f;                  // 2^-90
      if (top_v == 0.0f || top_m < 7.8886090522101181e-31f) top_m = 0.0f;  // 2^-100
      const float im = top_m > 0.0f ? __fdiv_rn(16129.0f, top_m) : 0.0f;
      const float iv = top_v > 0.0f ? __fdiv_rn(4228250625.0f, top_v) : 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t word = (e >> 2) + 32 * h;
        const u32x4 r = philox4x32_10(u32x4{(uint32_t)word, (uint32_t)(word >> 32), (uint32_t)step, kSaltAdam}, keys);
        const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
        uint32_t qm[4], qv[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 mk = m[h][k], s = mul2(mk, both(im));
          const float2 cm = codes_m(make_float2(fabsf(s.x), fabsf(s.y)), low_halves(rw[2 * k], rw[2 * k + 1]));
          const float2 cv = codes_v(product2(v[h][k], both(iv), a.minus_zero), high_halves(rw[2 * k], rw[2 * k + 1]), a.minus_zero);
          const float2 im8 = add2(make_float2(copysignf(cm.x, mk.x), copysignf(cm.y, mk.y)), both(12582912.0f));
          const float2 iv8 = add2(cv, both(12582912.0f));
          qm[2 * k] = __float_as_uint(im8.x), qm[2 * k + 1] = __float_as_uint(im8.y);
          qv[2 * k] = __float_as_uint(iv8.x), qv[2 * k + 1] = __float_as_uint(iv8.y);
        }
        *reinterpret_cast<uint32_t*>(reinterpret_cast<int8_t*>(a.m) + e + 128 * h) = pack4(qm[0], qm[1], qm[2], qm[3]);
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(a.v) + e + 128 * h) = pack4(qv[0], qv[1], qv[2], qv[3]);
      }
      if ((threadIdx.x & 31) == 0) {
        a.m_scale[e >> 8] = top_m;
        a.v_scale[e >> 8] = top_v;
      }
    }
  }
  if (!ready) {
    barrier();
    count();
  }
  if (threadIdx.x == 0 && a.last && before == gridDim.x - 1) {
    a.ctl->step = step;
    a.ctl->ticket = 0ull;
  }
}

// Values of codes: four elements per thread and step, four steps of 1024 elements on their way; 4096 elements a CTA, for short
// CTAs that follow each other keep the memory busier than loops (33.6 M: 58 us, 5.8 TB/s; 67 us with 8 CTAs an SM).
__global__ void __launch_bounds__(256)
    k_adamw_values(const int8_t* __restrict__ m, const uint8_t* __restrict__ v, const float* __restrict__ m_scale,
                   const float* __restrict__ v_scale, int64_t elements, float* __restrict__ mf, float* __restrict__ vf) {
  for (int64_t base = (int64_t)blockIdx.x * 4096; base < elements; base += (int64_t)gridDim.x * 4096) {
    uint32_t mc[4], vc[4];
    float um[4], uv[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int64_t e = base + s * 1024 + 4 * threadIdx.x;
      if (e < elements) {
        mc[s] = __ldg(reinterpret_cast<const uint32_t*>(m + e)) ^ 0x80808080u;
        vc[s] = __ldg(reinterpret_cast<const uint32_t*>(v + e));
        um[s] = __ldg(m_scale + (e >> 8)), uv[s] = __ldg(v_scale + (e >> 8));
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int64_t e = base + s * 1024 + 4 * threadIdx.x;
      if (e < elements) {
        const float x1 = __fmul_rn(um[s], 1.0f / 16129.0f), y1 = __fmul_rn(uv[s], 1.0f / 4228250625.0f);
        float x[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float c8 = __fsub_rn(byte_high(mc[s], k), 8388736.0f);
          x[k] = __fmul_rn(__fmul_rn(c8, fabsf(c8)), x1);
          y[k] = __fmul_rn(fourth(__fsub_rn(byte_high(vc[s], k), 8388608.0f)), y1);
        }
        *reinterpret_cast<float4*>(mf + e) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(vf + e) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
  }
}

// Whether the root that takes a subnormal v for 0 is near enough: what it loses, below 2^-63 / sqrt(1 - b2) of the denominator,
// is at most 2^-27 of eps.  With the default betas that holds from eps = 4.6e-10 on; roots of subnormal v take 141.6 us of
// 33.6 M weights, against 139.4.
bool flushes_roots(double eps, double beta2) { return eps * sqrt(1.0 - beta2) >= 1.4551915228366852e-11; }  // 2^-36

template <int BITS, int T, bool ROOTS>
int launch_adamw(const tthrml_adamw_tensor* t, int32_t n, AdamArgs a, int sms, cudaStream_t st) {
  AdamTable<T> tab;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    tab.t[i] = t[i];
    tab.first_chunk[i] = (int32_t)chunks;
    chunks += (t[i].n + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffff) {
      set_error("tthrml_adamw_step: too many elements for one launch");
      return TTHRML_ERR_ARG;
    }
  }
  tab.first_chunk[n] = (int32_t)chunks;
  a.n_tensors = n;
  // Two chunks a CTA, but no fewer CTAs than run at once: 33.6 M float32 weights took 142 us so, 149 with one chunk a CTA, 144
  // and 147 with three and six, 155 with 8 CTAs an SM; 600 tensors of 3.34 M bfloat16 weights 22.3, 23.0, 27.8 and 23.5, 21.9.
  const int64_t least = 4 * (int64_t)sms < chunks ? 4 * (int64_t)sms : chunks, want = (chunks + 1) / 2;
  const int grid = (int)(want > least ? want : least);
  k_adamw<BITS, T, ROOTS><<<grid, kAdamThreads, 0, st>>>(tab, a);
  return launch_status("k_adamw launch");
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_adamw_step(const tthrml_adamw_tensor* tensors_host, int64_t n_tensors, int32_t state_bits,
                                 void* exp_avg, void* exp_avg_sq, float* exp_avg_scale, float* exp_avg_sq_scale,
                                 tthrml_adamw_ctl* ctl, double beta1, double beta2, double eps, double weight_decay,
                                 uint64_t seed, void* stream) {
  using namespace tthrml;
  if (n_tensors == 0) return TTHRML_OK;
  if (!tensors_host || !exp_avg || !exp_avg_sq || !ctl || (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale))) {
    set_error("tthrml_adamw_step: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (state_bits != 8 && state_bits != 32) {
    set_error("tthrml_adamw_step: state_bits must be 8 or 32 (got %d)", (int)state_bits);
    return TTHRML_ERR_ARG;
  }
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-30) || !(weight_decay >= 0.0)) {
    set_error("tthrml_adamw_step: betas must lie in [0, 1), eps be at least 1e-30 and weight_decay not below 0");
    return TTHRML_ERR_ARG;
  }
  if (n_tensors < 0 || (uintptr_t)exp_avg % 16 || (uintptr_t)exp_avg_sq % 16) {
    set_error("tthrml_adamw_step: moments must be 16-byte aligned");
    return TTHRML_ERR_ARG;
  }
  for (int64_t i = 0; i < n_tensors; ++i) {
    const tthrml_adamw_tensor& t = tensors_host[i];
    const int64_t pb = dtype_bytes(t.param_dtype), gb = dtype_bytes(t.grad_dtype);
    if (t.n < 1 || !t.param || !t.grad || t.state < 0 || t.state % 256 || pb < 2 || gb < 2 ||
        ((uintptr_t)t.param & (pb - 1)) || ((uintptr_t)t.grad & (gb - 1))) {  // 2 or 4 bytes
      set_error("tthrml_adamw_step: tensor %lld: elements %lld, state offset %lld (a multiple of 256), types %d, %d",
                (long long)i, (long long)t.n, (long long)t.state, (int)t.param_dtype, (int)t.grad_dtype);
      return TTHRML_ERR_ARG;
    }
  }
  AdamArgs a;
  a.m = exp_avg;
  a.v = exp_avg_sq;
  a.m_scale = exp_avg_scale;
  a.v_scale = exp_avg_sq_scale;
  a.ctl = ctl;
  a.b1 = (float)beta1;
  a.d1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.d2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.minus_zero = -0.0f;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.weight_decay = weight_decay;
  a.seed = seed;
  int sms = 0, dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return cuda_status(e, "tthrml_adamw_step: device query");
  cudaStream_t st = (cudaStream_t)stream;
  constexpr int kMost = 700;  // 44 bytes each, within the 32764 bytes of a launch's parameters
  for (int64_t i = 0; i < n_tensors; i += kMost) {
    const int32_t n = (int32_t)(n_tensors - i < kMost ? n_tensors - i : kMost);
    a.last = i + n == n_tensors;
    // a launch copies its whole table: the smallest that holds the tensors (25 tensors: 8.6 us a step with the largest)
    const auto launch = [&](auto bits, auto roots) {
      constexpr int B = decltype(bits)::value;
      constexpr bool R = decltype(roots)::value;
      return n <= 24    ? launch_adamw<B, 24, R>(tensors_host + i, n, a, sms, st)
             : n <= 150 ? launch_adamw<B, 150, R>(tensors_host + i, n, a, sms, st)
                        : launch_adamw<B, kMost, R>(tensors_host + i, n, a, sms, st);
    };
    const int rc = state_bits == 32 ? launch(std::integral_constant<int, 32>{}, std::false_type{})
                   : flushes_roots(eps, beta2) ? launch(std::integral_constant<int, 8>{}, std::false_type{})
                                               : launch(std::integral_constant<int, 8>{}, std::true_type{});
    if (rc) return rc;
  }
  return TTHRML_OK;
}

extern "C" int tthrml_adamw_values(const int8_t* exp_avg, const uint8_t* exp_avg_sq, const float* exp_avg_scale,
                                   const float* exp_avg_sq_scale, int64_t elements, float* exp_avg_out,
                                   float* exp_avg_sq_out, void* stream) {
  using namespace tthrml;
  if (elements == 0) return TTHRML_OK;
  if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !exp_avg_out || !exp_avg_sq_out) {
    set_error("tthrml_adamw_values: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (elements < 0 || elements % 256 || (uintptr_t)exp_avg % 16 || (uintptr_t)exp_avg_sq % 16 ||
      (uintptr_t)exp_avg_out % 16 || (uintptr_t)exp_avg_sq_out % 16) {
    set_error("tthrml_adamw_values: elements must be a multiple of 256 and buffers 16-byte aligned (got %lld)",
              (long long)elements);
    return TTHRML_ERR_ARG;
  }
  const int64_t blocks = (elements + 4095) / 4096;
  k_adamw_values<<<(unsigned)(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, (cudaStream_t)stream>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, elements, exp_avg_out, exp_avg_sq_out);
  return launch_status("k_adamw_values launch");
}
