// 8-bit integer product for one or two rows (single tokens / chains), the rows quantised in the same launch:
//     y[m][n] = (sum_k q[m][k] w[n][k]) * (s_x[m] * s_w[n]) + bias[n].
//
// Bound: the weights are read once (N K bytes); there is nothing to reuse them for, so the tensor cores are left
// alone.  Every CTA quantises the rows itself into shared memory (M K elements from L2; a launch of its own would cost
// more than that), while the first weight vectors are already on their way.  The multiplications are dp4a (exact in int32
// for K <= 131071), whose rate is what ends this form.  One and two rows, and three (on the tensor cores) beside them, replayed
// from a graph: K = 1000, N = 3000 in 3.3, 3.7 and 6.4 us; 4096, 8192 in 7.0, 8.8 and 9.4 with the weights in L2, 9.4, 10.4
// and 11.9 with weights that take turns; 8192, 4096 in 8.0, 10.7 and 9.2, or 10.3, 12.2 and 11.8.
#include "int8_common.cuh"

namespace tthrml {
namespace {

struct FewArgs {
  const void* x;         // [M][x_ld] elements of the input type
  int64_t x_ld;
  const float* x_scale;  // [M], 8-bit input only; NULL: ones
  const int8_t* w;       // [N][w_pitch]
  int64_t w_pitch;
  const float* w_scale;  // [N]
  const float* bias;     // [N] or NULL
  void* out;             // [M][out_ld] elements of the output type
  int64_t out_ld;
  int32_t out_dtype;
  int32_t M, K;
  int64_t N;
};

constexpr int kFewThreads = 256, kFewWarps = 8;
constexpr int kFewSmemMax = TTHRML_INT8_FEW_BYTES;

__device__ __forceinline__ void store_out(void* out, int32_t dtype, int64_t at, float v) {
  if (dtype == TTHRML_DT_F32)
    reinterpret_cast<float*>(out)[at] = v;
  else if (dtype == TTHRML_DT_BF16)
    reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
}

// The 16 weights from column k of a row of K (the row start is 16-byte aligned); zeros behind the end.
__device__ __forceinline__ uint4 weights16(const int8_t* row, int64_t k, int64_t K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) v[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Quantises rows of x into xs (pitch kp, zero-padded): all eight warps take one row, four each of two.
template <typename T, int MP>
__device__ __forceinline__ void quantize_into(const FewArgs& a, int8_t* xs, int kp, float* sxs, uint32_t* part) {
  constexpr int kGroup = kFewWarps / MP;  // warps per row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m = warp / kGroup, t = (warp % kGroup) * 32 + lane;
  const T* xr = reinterpret_cast<const T*>(a.x) + (int64_t)(m < a.M ? m : 0) * a.x_ld;
  const bool vectors = (uintptr_t)xr % 16 == 0;
  const int K = m < a.M ? a.K : 0;
  float most = 0.0f;
  for (int c = 8 * t; c < K; c += 256 * kGroup) {
    float f[8];
    if (vectors && c + 8 <= K) {
      unpack8(load8(xr + c), f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i < K ? to_f32(xr[c + i]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_abs(most, f[i]);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(most));
  if (lane == 0) part[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGroup; ++i) top = max(top, part[m * kGroup + i]);
  const RowScale s = row_scale(top);
  if (t == 0) sxs[m] = s.scale;
  for (int c = 8 * t; c < kp; c += 256 * kGroup) {
    float f[8];
    if (vectors && c + 8 <= K) {
      unpack8(load8(xr + c), f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i < K ? to_f32(xr[c + i]) : 0.0f;
    }
    *reinterpret_cast<uint2*>(xs + m * kp + c) = quantize8(f, s.inv);
  }
}

// Each warp walks over units, a unit of the weights at a time, kVecs 16-byte vectors per lane and step; the next step's
// vectors are on their way while the current ones are multiplied, so four CTAs of eight warps keep 64 KB of weights on
// their way to an SM.  33.5 M weights and one row took 9.0 us so, 10.4 us with two CTAs and eight vectors, 9.8 and 10.1 us
// with three and five CTAs of four vectors, 11.5 us with six of two.
constexpr int kVecs = 4, kFewCtas = 4;

template <typename T, int MP>
__global__ void __launch_bounds__(kFewThreads, kFewCtas) k_int8_few(FewArgs a) {
  extern __shared__ __align__(16) int8_t xs[];
  __shared__ float sxs[8];
  __shared__ uint32_t part[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kp = (a.K + 15) & ~15;
  const int64_t stride = (int64_t)gridDim.x * kFewWarps;
  int64_t n = (int64_t)warp * gridDim.x + blockIdx.x;  // the last, partial round of units is spread over the CTAs
  uint4 next[kVecs];
  auto fetch = [&](int64_t unit, int k0) {
    const int8_t* row = a.w + unit * a.w_pitch;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int k = k0 + (u * 32 + lane) * 16;
      next[u] = k < a.K ? weights16(row, k, a.K) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  if (n < a.N) fetch(n, 0);
  if constexpr (sizeof(T) == 1) {
    const int8_t* x = reinterpret_cast<const int8_t*>(a.x);
    for (int m = 0; m < MP; ++m) {
      for (int c = threadIdx.x; c < kp; c += kFewThreads) xs[m * kp + c] = m < a.M && c < a.K ? x[m * a.x_ld + c] : (int8_t)0;
    }
    if (threadIdx.x < MP) sxs[threadIdx.x] = (int)threadIdx.x < a.M && a.x_scale ? a.x_scale[threadIdx.x] : 1.0f;
  } else {
    quantize_into<T, MP>(a, xs, kp, sxs, part);
  }
  __syncthreads();
  int32_t acc[MP];
#pragma unroll
  for (int m = 0; m < MP; ++m) acc[m] = 0;
  for (int k0 = 0; n < a.N;) {
    uint4 cur[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) cur[u] = next[u];
    const int64_t unit = n;
    const int base = k0;
    k0 += kVecs * 512;
    if (k0 >= a.K) {
      k0 = 0;
      n += stride;
    }
    if (n < a.N) fetch(n, k0);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int k = base + (u * 32 + lane) * 16;
      if (k < a.K) {
#pragma unroll
        for (int m = 0; m < MP; ++m) {
          const int4 q = *reinterpret_cast<const int4*>(xs + m * kp + k);
          acc[m] = __dp4a((int)cur[u].x, q.x, acc[m]);
          acc[m] = __dp4a((int)cur[u].y, q.y, acc[m]);
          acc[m] = __dp4a((int)cur[u].z, q.z, acc[m]);
          acc[m] = __dp4a((int)cur[u].w, q.w, acc[m]);
        }
      }
    }
    if (k0 == 0) {  // the unit's last step
#pragma unroll
      for (int m = 0; m < MP; ++m) {
        const int32_t sum = __reduce_add_sync(0xffffffffu, acc[m]);
        acc[m] = 0;
        if (lane == m && m < a.M) {
          float y = __fmul_rn((float)sum, __fmul_rn(sxs[m], __ldg(a.w_scale + unit)));
          if (a.bias) y = __fadd_rn(y, __ldg(a.bias + unit));
          store_out(a.out, a.out_dtype, m * a.out_ld + unit, y);
        }
      }
    }
  }
}

template <typename T, int MP>
int launch_few(const FewArgs& a, cudaStream_t st) {
  const int smem = MP * ((a.K + 15) & ~15);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return cuda_status(e, "tthrml_int8_product_few: device query");
  const int64_t want = (a.N + kFewWarps - 1) / kFewWarps, fit = 224 * 1024 / (smem + 2048);
  const int64_t most = (int64_t)sms * (fit < 1 ? 1 : (fit > kFewCtas ? kFewCtas : fit));
  const int64_t grid = want < most ? want : most;
  // The 48 KiB of a launch without the attribute hold the kernel's static shared memory too (64 bytes).  The attribute is per
  // device and function; setting it again is cheap.
  if (smem > 47 * 1024) {
    e = cudaFuncSetAttribute(k_int8_few<T, MP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmemMax);
    if (e != cudaSuccess) return cuda_status(e, "k_int8_few shared memory attribute");
  }
  k_int8_few<T, MP><<<(unsigned)grid, kFewThreads, smem, st>>>(a);
  return launch_status("k_int8_few launch");
}

template <typename T>
int launch_few_rows(const FewArgs& a, cudaStream_t st) {
  return a.M == 1 ? launch_few<T, 1>(a, st) : launch_few<T, 2>(a, st);
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_int8_product_few(const void* x, int32_t x_dtype, int64_t x_ld, const float* x_scale,
                                       const int8_t* weights, int64_t w_pitch, const float* w_scale, int64_t rows,
                                       int64_t units, int64_t cols, const float* bias, void* out, int32_t out_dtype,
                                       int64_t out_ld, void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  if (!x || !weights || !w_scale || !out) {
    set_error("tthrml_int8_product_few: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (rows < 1 || rows > 2 || units < 1 || cols < 1 || cols > TTHRML_INT8_MAX_COLS || units > 0x3fffffffLL) {
    set_error("tthrml_int8_product_few: 1 or 2 rows and 1 to %d columns (got %lld rows, %lld units, %lld columns)",
              TTHRML_INT8_MAX_COLS, (long long)rows, (long long)units, (long long)cols);
    return TTHRML_ERR_ARG;
  }
  if (rows * ((cols + 15) / 16 * 16) > kFewSmemMax) {
    set_error("tthrml_int8_product_few: %lld rows of %lld columns exceed the shared memory that holds them",
              (long long)rows, (long long)cols);
    return TTHRML_ERR_ARG;
  }
  if (dtype_bytes(x_dtype) == 0 || out_dtype == TTHRML_DT_I8 || dtype_bytes(out_dtype) == 0) {
    set_error("tthrml_int8_product_few: unknown element type (input code %d, output code %d)", (int)x_dtype,
              (int)out_dtype);
    return TTHRML_ERR_ARG;
  }
  if ((uintptr_t)weights % 16 || w_pitch % 16 || w_pitch < cols || (x_ld < cols && rows > 1) || out_ld < units) {
    set_error("tthrml_int8_product_few: weights must be 16-byte aligned with a pitch >= cols that is a multiple of "
              "16, and rows must not overlap (got pitches %lld, %lld, %lld)", (long long)w_pitch, (long long)x_ld,
              (long long)out_ld);
    return TTHRML_ERR_ARG;
  }
  FewArgs a;
  a.x = x;
  a.x_ld = x_ld;
  a.x_scale = x_scale;
  a.w = weights;
  a.w_pitch = w_pitch;
  a.w_scale = w_scale;
  a.bias = bias;
  a.out = out;
  a.out_ld = out_ld;
  a.out_dtype = out_dtype;
  a.M = (int32_t)rows;
  a.K = (int32_t)cols;
  a.N = units;
  cudaStream_t st = (cudaStream_t)stream;
  switch (x_dtype) {
    case TTHRML_DT_F32: return launch_few_rows<float>(a, st);
    case TTHRML_DT_BF16: return launch_few_rows<__nv_bfloat16>(a, st);
    case TTHRML_DT_F16: return launch_few_rows<__half>(a, st);
    default: return launch_few_rows<int8_t>(a, st);
  }
}
