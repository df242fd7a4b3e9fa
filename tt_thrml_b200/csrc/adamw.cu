// AdamW (Adam with decoupled weight decay; Loshchilov and Hutter, ICLR 2019) over many tensors in one launch:
//     m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//     p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with the moments in float32 or in 8-bit codes.  All arithmetic is float32, every operation rounded by itself.
//
// Bound: memory.  Each element of the tensors and moments is read once and written once: 2 p + g + 16 bytes with
// float32 moments, 2 p + g + 4 + 1/16 with codes (p, g: bytes of a parameter and a gradient).
//
// The tensors' addresses travel in the launch's parameters, so a step uploads nothing and a captured graph keeps its
// own copy.  The moments of all tensors lie in one buffer, each tensor's segment padded to 256 elements.  A CTA takes a
// contiguous range of 2048-element chunks of the concatenated tensors (a chunk never spans two tensors); a thread
// holds eight consecutive elements.  The step counter and the learning rate stand in device memory, so a replayed
// graph counts on; the last CTA of a step's last launch advances the counter.
//
// 8-bit codes, one warp per block of 256 elements with the block's largest |m| and v as scales:
//     m = sign q^2 max|m| / 127^2, q = 0..127;      v = q^4 max v / 255^4, q = 0..255.
// The powers give small values small steps: v spans 255^4 = 2^32, that is 2^16 in gradient magnitude.  A value is
// rounded to the code below or above at random with the probability that keeps its mean, because a code's step exceeds
// what one step of the averages changes ((1 - b2) = 0.1 % of v): rounding to nearest would hold them where they are.
// The random words are Philox4x32-10 at (element / 4, element / 4 >> 32, step, "ADMW"), word element % 4, low half
// for m and high half for v, so a run can be repeated.  A v > 0 is never rounded to zero, or m / (0 + eps) would
// follow.  A block whose largest v is below 2^-90 is held as zeros; one that takes in an infinity or a NaN is NaN.
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
  double beta1, beta2, weight_decay;
  uint64_t seed;
  int32_t n_tensors;
  int32_t last;     // this launch ends the step
};

template <typename T>
__device__ __forceinline__ void load_elems(const void* base, int64_t i, int64_t n, bool vectors, float (&f)[8]) {
  const T* p = reinterpret_cast<const T*>(base) + i;
  if (vectors && i + 8 <= n) {
    Vec8<T> v;
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 2); ++k) v.w[k] = *(reinterpret_cast<const uint4*>(p) + k);
    unpack8(v, f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = i + k < n ? to_f32(p[k]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_elems(void* base, int64_t i, int64_t n, bool vectors, const float (&f)[8]) {
  T* p = reinterpret_cast<T*>(base) + i;
  if (vectors && i + 8 <= n) {
    Vec8<T> v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = from_f32<T>(f[k]);
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 2); ++k) *(reinterpret_cast<uint4*>(p) + k) = v.w[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[k] = from_f32<T>(f[k]);
  }
}
__device__ __forceinline__ void load_any(int32_t dtype, const void* base, int64_t i, int64_t n, bool vectors, float (&f)[8]) {
  if (dtype == TTHRML_DT_F32)
    load_elems<float>(base, i, n, vectors, f);
  else if (dtype == TTHRML_DT_BF16)
    load_elems<__nv_bfloat16>(base, i, n, vectors, f);
  else
    load_elems<__half>(base, i, n, vectors, f);
}
__device__ __forceinline__ void store_any(int32_t dtype, void* base, int64_t i, int64_t n, bool vectors, const float (&f)[8]) {
  if (dtype == TTHRML_DT_F32)
    store_elems<float>(base, i, n, vectors, f);
  else if (dtype == TTHRML_DT_BF16)
    store_elems<__nv_bfloat16>(base, i, n, vectors, f);
  else
    store_elems<__half>(base, i, n, vectors, f);
}

// Byte j of a word as a float, unsigned: the byte under the exponent of 2^23, which is subtracted.
__device__ __forceinline__ float byte_f32(uint32_t w, int j) {
  return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540u | (uint32_t)j)), 8388608.0f);
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// floor of 0 <= x < 2^22, one too few at odd integers (x - 1/2 is a tie there, rounded to even)
__device__ __forceinline__ float near_floor(float x) {
  return __fsub_rn(__fadd_rn(__fsub_rn(x, 0.5f), 12582912.0f), 12582912.0f);
}
// h + 1/2 of a half word h: 65536 times a uniform that is never 0 or 1
__device__ __forceinline__ float low_half(uint32_t w) {
  return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7410u)), 8388607.5f);
}
__device__ __forceinline__ float high_half(uint32_t w) {
  return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7432u)), 8388607.5f);
}

// Code of y = m 127^2 / max|m| >= 0: the largest k with k^2 <= y, or k + 1 with probability (y - k^2) / (2 k + 1).  The
// approximate root is off by one only next to a whole number; u65536 is 65536 u, and the powers of two are exact.
__device__ __forceinline__ float code_m(float y, float u65536) {
  float k = near_floor(sqrt_approx(y));
  float k2 = __fmul_rn(k, k), span = __fadd_rn(__fadd_rn(k, k), 1.0f);
  float over = __fsub_rn(y, k2);
  if (over < 0.0f || over >= span) {
    k = over < 0.0f ? __fsub_rn(k, 1.0f) : __fadd_rn(k, 1.0f);
    k2 = __fmul_rn(k, k);
    span = __fadd_rn(__fadd_rn(k, k), 1.0f);
    over = __fsub_rn(y, k2);
  }
  const float q = __fmul_rn(u65536, span) < __fmul_rn(over, 65536.0f) ? __fadd_rn(k, 1.0f) : k;
  return fminf(q, 127.0f);
}
__device__ __forceinline__ float fourth(float k) {
  const float k2 = __fmul_rn(k, k);
  return __fmul_rn(k2, k2);
}
// Code of y = v 255^4 / max v >= 0, likewise with fourth powers; a y > 0 gets at least 1.
__device__ __forceinline__ float code_v(float y, float u65536) {
  float k = near_floor(sqrt_approx(sqrt_approx(y)));
  float k4 = fourth(k), n4 = fourth(__fadd_rn(k, 1.0f));
  if (k4 > y || n4 <= y) {
    k = k4 > y ? __fsub_rn(k, 1.0f) : __fadd_rn(k, 1.0f);
    k4 = fourth(k);
    n4 = fourth(__fadd_rn(k, 1.0f));
  }
  const float span = __fsub_rn(n4, k4), over = __fsub_rn(y, k4);
  float q = __fmul_rn(u65536, span) < __fmul_rn(over, 65536.0f) ? __fadd_rn(k, 1.0f) : k;
  if (k == 0.0f) q = y > 0.0f ? 1.0f : 0.0f;
  return fminf(q, 255.0f);
}
// Low byte of the integer held by a float in -2^22 .. 2^22.
__device__ __forceinline__ uint32_t int_byte(float q) { return __float_as_uint(__fadd_rn(q, 12582912.0f)); }
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}

template <int BITS, int T>
__global__ void __launch_bounds__(kAdamThreads)
    k_adamw(const __grid_constant__ AdamTable<T> tab, const __grid_constant__ AdamArgs a) {
  __shared__ float coef[4];  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd, step
  const int chunks = tab.first_chunk[a.n_tensors];
  const int c_first = (int)((int64_t)chunks * blockIdx.x / gridDim.x);
  const int c_last = (int)((int64_t)chunks * (blockIdx.x + 1) / gridDim.x);
  const int64_t step = a.ctl->step + 1;
  if (threadIdx.x == 0) {
    const double lr = a.ctl->lr, t = (double)step;
    coef[0] = (float)(lr / (1.0 - pow(a.beta1, t)));
    coef[1] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, t)));
    coef[2] = (float)(1.0 - lr * a.weight_decay);
  }
  __syncthreads();
  const float step_size = coef[0], r_bias2 = coef[1], keep = coef[2];
  const PhiloxKeys keys = philox_keys((uint32_t)a.seed, (uint32_t)(a.seed >> 32));
  int ti = 0;
  for (int lo = 0, hi = a.n_tensors; hi - lo > 1;) {  // the tensor of the first chunk
    const int mid = (lo + hi) >> 1;
    (tab.first_chunk[mid] <= c_first ? lo : hi) = mid;
    ti = lo;
  }
  for (int c = c_first; c < c_last; ++c) {
    while (tab.first_chunk[ti + 1] <= c) ++ti;
    const tthrml_adamw_tensor& t = tab.t[ti];
    const int64_t i = (int64_t)(c - tab.first_chunk[ti]) * kChunk + 8 * threadIdx.x;
    const int64_t padded = (t.n + 255) & ~(int64_t)255;
    if (i >= padded) continue;  // whole warps: a warp covers 256 elements
    const int64_t e = t.state + i;
    const bool pv = (uintptr_t)t.param % 16 == 0, gv = (uintptr_t)t.grad % 16 == 0;
    float p[8], g[8], m[8], v[8];
    load_any(t.grad_dtype, t.grad, i, t.n, gv, g);
    load_any(t.param_dtype, t.param, i, t.n, pv, p);
    if (BITS == 32) {
      const float4* mp = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.m) + e);
      const float4* vp = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.v) + e);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 x = mp[k], y = vp[k];
        m[4 * k] = x.x, m[4 * k + 1] = x.y, m[4 * k + 2] = x.z, m[4 * k + 3] = x.w;
        v[4 * k] = y.x, v[4 * k + 1] = y.y, v[4 * k + 2] = y.z, v[4 * k + 3] = y.w;
      }
    } else {
      const uint2 mc = *reinterpret_cast<const uint2*>(reinterpret_cast<const int8_t*>(a.m) + e);
      const uint2 vc = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.v) + e);
      const float um = __fmul_rn(a.m_scale[e >> 8], 1.0f / 16129.0f), uv = __fmul_rn(a.v_scale[e >> 8], 1.0f / 4228250625.0f);
      const uint32_t mw[2] = {mc.x ^ 0x80808080u, mc.y ^ 0x80808080u}, vw[2] = {vc.x, vc.y};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float c8 = __fsub_rn(byte_f32(mw[k >> 2], k & 3), 128.0f);
        m[k] = __fmul_rn(__fmul_rn(c8, fabsf(c8)), um);
        v[k] = __fmul_rn(fourth(byte_f32(vw[k >> 2], k & 3)), uv);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = __fadd_rn(__fmul_rn(m[k], a.b1), __fmul_rn(g[k], a.d1));
      v[k] = __fadd_rn(__fmul_rn(v[k], a.b2), __fmul_rn(__fmul_rn(g[k], g[k]), a.d2));
      if (BITS == 32) {
        const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v[k]), r_bias2), a.eps);
        p[k] = __fsub_rn(__fmul_rn(p[k], keep), __fmul_rn(__fdiv_rn(m[k], denom), step_size));
      } else {
        // the hardware's root and quotient (2^-21 of the update at most, whose moments are codes to about 1 %): the step on
        // codes is bound by its instructions
        const float denom = __fadd_rn(__fmul_rn(sqrt_approx(v[k]), r_bias2), a.eps);
        p[k] = __fsub_rn(__fmul_rn(p[k], keep), __fmul_rn(__fdividef(m[k], denom), step_size));
      }
    }
    store_any(t.param_dtype, t.param, i, t.n, pv, p);
    if (BITS == 32) {
      float4* mp = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.m) + e);
      float4* vp = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.v) + e);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mp[k] = make_float4(m[4 * k], m[4 * k + 1], m[4 * k + 2], m[4 * k + 3]);
        vp[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
    } else {
      uint32_t tm = 0u, tv = 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        tm = max(tm, abs_bits(m[k]));
        tv = max(tv, abs_bits(v[k]));
      }
      tm = __reduce_max_sync(0xffffffffu, tm);
      tv = __reduce_max_sync(0xffffffffu, tv);
      float top_m = __uint_as_float(tm), top_v = __uint_as_float(tv);
      const bool finite = tm < 0x7F800000u && tv < 0x7F800000u;
      if (!finite) top_m = top_v = __uint_as_float(0x7FC00000u);
      if (top_v < 8.0779356694631609e-28f) top_v = 0.0f;                  // 2^-90
      if (top_v == 0.0f || top_m < 7.8886090522101181e-31f) top_m = 0.0f;  // 2^-100
      const float im = top_m > 0.0f ? __fdiv_rn(16129.0f, top_m) : 0.0f;
      const float iv = top_v > 0.0f ? __fdiv_rn(4228250625.0f, top_v) : 0.0f;
      uint32_t qm[8], qv[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t word = (e >> 2) + h;
        const u32x4 r = philox4x32_10(u32x4{(uint32_t)word, (uint32_t)(word >> 32), (uint32_t)step, kSaltAdam}, keys);
        const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = 4 * h + j;
          const float q = code_m(__fmul_rn(fabsf(m[k]), im), low_half(rw[j]));
          qm[k] = int_byte(copysignf(q, m[k]));
          qv[k] = int_byte(code_v(__fmul_rn(v[k], iv), high_half(rw[j])));
        }
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<int8_t*>(a.m) + e) =
          make_uint2(pack_bytes(qm[0], qm[1], qm[2], qm[3]), pack_bytes(qm[4], qm[5], qm[6], qm[7]));
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.v) + e) =
          make_uint2(pack_bytes(qv[0], qv[1], qv[2], qv[3]), pack_bytes(qv[4], qv[5], qv[6], qv[7]));
      if ((threadIdx.x & 31) == 0) {
        a.m_scale[e >> 8] = top_m;
        a.v_scale[e >> 8] = top_v;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && a.last) {
    __threadfence();
    if (atomicAdd(&a.ctl->ticket, 1ull) == gridDim.x - 1) {  // every CTA has read the step
      a.ctl->step = step;
      a.ctl->ticket = 0ull;
    }
  }
}

__global__ void __launch_bounds__(256)
    k_adamw_values(const int8_t* __restrict__ m, const uint8_t* __restrict__ v, const float* __restrict__ m_scale,
                   const float* __restrict__ v_scale, int64_t elements, float* __restrict__ mf, float* __restrict__ vf) {
  for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; e < elements; e += (int64_t)gridDim.x * 2048) {
    const uint2 mc = *reinterpret_cast<const uint2*>(m + e), vc = *reinterpret_cast<const uint2*>(v + e);
    const float um = __fmul_rn(m_scale[e >> 8], 1.0f / 16129.0f), uv = __fmul_rn(v_scale[e >> 8], 1.0f / 4228250625.0f);
    const uint32_t mw[2] = {mc.x ^ 0x80808080u, mc.y ^ 0x80808080u}, vw[2] = {vc.x, vc.y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[4], y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float c8 = __fsub_rn(byte_f32(mw[h], k), 128.0f);
        x[k] = __fmul_rn(__fmul_rn(c8, fabsf(c8)), um);
        y[k] = __fmul_rn(fourth(byte_f32(vw[h], k)), uv);
      }
      reinterpret_cast<float4*>(mf + e)[h] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(vf + e)[h] = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
}

template <int BITS, int T>
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
  const int64_t want = 4 * (int64_t)sms;
  const int grid = (int)(chunks < want ? (chunks > 0 ? chunks : 1) : want);
  k_adamw<BITS, T><<<grid, kAdamThreads, 0, st>>>(tab, a);
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
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps > 0.0) || !(weight_decay >= 0.0)) {
    set_error("tthrml_adamw_step: betas must lie in [0, 1), eps above 0 and weight_decay not below 0");
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
        (uintptr_t)t.param % pb || (uintptr_t)t.grad % gb) {
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
    int rc;
    if (state_bits == 32)
      rc = n <= 24 ? launch_adamw<32, 24>(tensors_host + i, n, a, sms, st) : launch_adamw<32, kMost>(tensors_host + i, n, a, sms, st);
    else
      rc = n <= 24 ? launch_adamw<8, 24>(tensors_host + i, n, a, sms, st) : launch_adamw<8, kMost>(tensors_host + i, n, a, sms, st);
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
  const int64_t blocks = (elements + 2047) / 2048;
  k_adamw_values<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, (cudaStream_t)stream>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, elements, exp_avg_out, exp_avg_sq_out);
  return launch_status("k_adamw_values launch");
}
