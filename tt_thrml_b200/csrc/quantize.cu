// Rows to 8-bit integers with one float32 scale per row (the formula stands in int8_common.cuh).
//
// One pass over the input: each row is read once, kept in registers while its largest magnitude is reduced, and
// written as packed bytes.  Bound: memory (b read + 1 written byte per element).
//   k_quantize_rows<T, W>: W warps per row, as few as hold it in registers (1024 elements a warp, at most 8 warps), so that
//     a thread has four (float32: eight) 16-byte loads on their way: 8192 x 4096 bfloat16 took 41 us with eight warps a
//     row and half of their vectors empty.  Rows that do not start on 16 bytes are read as aligned vectors and shifted.
//     Longer rows read their tail again.
//   k_quantize_cols<T>: rows whose consecutive elements are strided but whose neighbours are adjacent (a transposed
//     matrix): a cluster of eight CTAs takes 32 rows, an eighth of the columns each; the lanes run along the rows.  A share
//     that fits stays in shared memory between the maximum, which the CTAs exchange, and the rounding.
#include "row_reader.cuh"
#include "tc_common.cuh"

namespace tthrml {
namespace {

// The quantised bytes of a vector.
template <typename T>
__device__ __forceinline__ void store_vector(int8_t* q, const Vec8<T>& v, float inv) {
  float f[8];
  unpack8(v, f);
  *reinterpret_cast<uint2*>(q) = quantize8(f, inv);
}

template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(256, 4)
    k_quantize_rows(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int contiguous,
                    int8_t* __restrict__ q, int64_t pitch, float* __restrict__ scale) {
  __shared__ uint32_t part[8];
  let_next_kernel_start();
  constexpr int kKept = 4, kStep = 32 * W * 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (int)threadIdx.x & (32 * W - 1);
  const int64_t row = (int64_t)blockIdx.x * (8 / W) + warp / W;
  const bool live = row < rows;
  if (!live) cols = pitch = 0;
  const T* xr = x + (live ? row : 0) * rs;
  const uint32_t off = (uint32_t)((uintptr_t)xr & 15u);
  const RowReader<T, ALIGNED> in = {xr, (int32_t)cols, cs, contiguous ? (off ? kShifted : kAligned) : kElements, off};
  Vec8<T> kept[kKept];
  MaxOf<T> most;
#pragma unroll
  for (int v = 0; v < kKept; ++v) kept[v] = in.vector(v * kStep + 8 * t);
#pragma unroll
  for (int v = 0; v < kKept; ++v) add_vector<T>(most, kept[v]);
  for (int64_t c = (int64_t)kKept * kStep + 8 * t; c < cols; c += kStep) add_vector<T>(most, in.vector((int32_t)c));
  uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(most.value()));
  if (W > 1) {
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, part[warp / W * W + i]);
  }
  const RowScale s = row_scale(top);
  if (live && t == 0) scale[row] = s.scale;
  int8_t* qr = q + row * pitch;  // pitch is a multiple of 16; columns from cols to pitch are written as zeros
#pragma unroll
  for (int v = 0; v < kKept; ++v) {
    const int64_t c = (int64_t)v * kStep + 8 * t;
    if (c < pitch) store_vector<T>(qr + c, kept[v], s.inv);
  }
  for (int64_t c = (int64_t)kKept * kStep + 8 * t; c < pitch; c += kStep) store_vector<T>(qr + c, in.vector((int32_t)c), s.inv);
}

// Rows adjacent in memory (row stride 1): lane = row, warp w takes columns w, w + 8, ... of the CTA's share.
constexpr int kColsCluster = 8, kColsKept = 512;  // columns of a share that shared memory keeps

template <typename T>
__global__ void __launch_bounds__(256)
    k_quantize_cols(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t cs, int8_t* __restrict__ q,
                    int64_t pitch, int64_t share, float* __restrict__ scale) {
  extern __shared__ __align__(16) unsigned char kept_raw[];
  T* kept = reinterpret_cast<T*>(kept_raw);  // [share][32] where it fits
  __shared__ uint32_t part[8][32];
  __shared__ uint32_t mine[32];
  __shared__ __align__(16) int8_t tile[32][144];  // 128 columns of 32 rows; the pitch spreads the rows over the banks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = (int)cluster_ctarank();
  const int64_t r0 = (int64_t)(blockIdx.x / kColsCluster) * 32, row = r0 + lane;
  const int64_t first = share * rank, last = first + share < pitch ? first + share : pitch;  // multiples of 16
  const bool fits = share <= kColsKept;
  const T* xr = x + (row < rows ? row : 0);
  const T zero = from_f32<T>(0.0f);
  uint32_t top = 0u;
#pragma unroll 8
  for (int64_t c = first + warp; c < last; c += 8) {
    const T v = row < rows && c < cols ? __ldg(xr + c * cs) : zero;
    if (fits) kept[(c - first) * 32 + lane] = v;
    top = max(top, abs_bits(to_f32(v)));
  }
  part[warp][lane] = top;
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, part[i][lane]);
    mine[lane] = top;
  }
  cluster_sync_all();
  top = 0u;
#pragma unroll
  for (int r = 0; r < kColsCluster; ++r) {
    uint32_t remote, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(&mine[lane])), "r"(r));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    top = max(top, v);
  }
  cluster_sync_all();  // every CTA has read the maxima before any leaves
  const RowScale s = row_scale(top);
  if (rank == 0 && warp == 0 && row < rows) scale[row] = s.scale;
  for (int64_t c0 = first; c0 < last; c0 += 128) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t c = c0 + warp + 8 * i;
      T v = zero;
      if (c < last) v = fits ? kept[(c - first) * 32 + lane] : (row < rows && c < cols ? __ldg(xr + c * cs) : zero);
      tile[lane][warp + 8 * i] = (int8_t)(quantize_low(to_f32(v), s.inv) & 255u);
    }
    __syncthreads();
    const int r = threadIdx.x >> 3, b = (threadIdx.x & 7) * 16;  // 32 rows x 8 vectors of 16 bytes
    if (r0 + r < rows && c0 + b < last)
      *reinterpret_cast<uint4*>(q + (r0 + r) * pitch + c0 + b) = *reinterpret_cast<const uint4*>(&tile[r][b]);
    __syncthreads();
  }
}

// int8 to bfloat16, 16 elements per thread (spins as operands of 16-bit products).
__global__ void __launch_bounds__(256) k_widen(const int8_t* __restrict__ src, __nv_bfloat16* __restrict__ dst, int64_t n) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16; i < n; i += (int64_t)gridDim.x * 4096) {
    if (i + 16 <= n) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + i));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t pair = w[k >> 1] >> (16 * (k & 1));
        const __nv_bfloat162 h = __floats2bfloat162_rn((float)(int8_t)(pair & 255u), (float)(int8_t)((pair >> 8) & 255u));
        o[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
      uint4* d = reinterpret_cast<uint4*>(dst + i);
      d[0] = make_uint4(o[0], o[1], o[2], o[3]);
      d[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      for (int64_t k = i; k < n; ++k) dst[k] = __float2bfloat16_rn((float)src[k]);
    }
  }
}

template <typename T>
int launch_quantize(const T* x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int8_t* q, int64_t pitch,
                    float* scale, cudaStream_t st) {
  if (cs != 1 && rs == 1) {
    int64_t share = (pitch / 16 + kColsCluster - 1) / kColsCluster * 16;
    const int smem = share <= kColsKept ? (int)(share * 32 * sizeof(T)) : 0;
    void* params[8] = {(void*)&x, (void*)&rows, (void*)&cols, (void*)&cs, (void*)&q, (void*)&pitch, (void*)&share, (void*)&scale};
    return launch_clusters((const void*)k_quantize_cols<T>, (unsigned)((rows + 31) / 32 * kColsCluster), kColsCluster, 256,
                           smem, params, st, "k_quantize_cols launch");
  }
  const int contiguous = cs == 1;
  const bool aligned = contiguous && (uintptr_t)x % 16 == 0 && (rs * (int64_t)sizeof(T)) % 16 == 0;
  const int warps = cols <= 1024 ? 1 : (cols <= 2048 ? 2 : (cols <= 4096 ? 4 : 8));
  const unsigned grid = (unsigned)((rows + 8 / warps - 1) / (8 / warps));
  const auto run = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(x, rows, cols, rs, cs, contiguous, q, pitch, scale); };
  if (warps == 1)
    aligned ? run(k_quantize_rows<T, 1, true>) : run(k_quantize_rows<T, 1, false>);
  else if (warps == 2)
    aligned ? run(k_quantize_rows<T, 2, true>) : run(k_quantize_rows<T, 2, false>);
  else if (warps == 4)
    aligned ? run(k_quantize_rows<T, 4, true>) : run(k_quantize_rows<T, 4, false>);
  else
    aligned ? run(k_quantize_rows<T, 8, true>) : run(k_quantize_rows<T, 8, false>);
  return launch_status("k_quantize_rows launch");
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_quantize_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                    int64_t col_stride, int8_t* values, int64_t pitch, float* scale, void* stream) {
  using namespace tthrml;
  if (rows == 0) return TTHRML_OK;
  if (!x || !values || !scale) {
    set_error("tthrml_quantize_rows: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (rows < 0 || cols < 1 || rows > 0x0fffffffLL || row_stride < 0 || col_stride < 1) {
    set_error("tthrml_quantize_rows: sizes and strides out of range (rows %lld, cols %lld, strides %lld, %lld)",
              (long long)rows, (long long)cols, (long long)row_stride, (long long)col_stride);
    return TTHRML_ERR_ARG;
  }
  if (pitch < cols || pitch % 16 || (uintptr_t)values % 16) {
    set_error("tthrml_quantize_rows: values must be 16-byte aligned with a pitch >= cols that is a multiple of 16 "
              "(got pitch %lld for %lld columns)", (long long)pitch, (long long)cols);
    return TTHRML_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case TTHRML_DT_F32:
      return launch_quantize((const float*)x, rows, cols, row_stride, col_stride, values, pitch, scale, st);
    case TTHRML_DT_BF16:
      return launch_quantize((const __nv_bfloat16*)x, rows, cols, row_stride, col_stride, values, pitch, scale, st);
    case TTHRML_DT_F16:
      return launch_quantize((const __half*)x, rows, cols, row_stride, col_stride, values, pitch, scale, st);
    default:
      set_error("tthrml_quantize_rows: input type must be float32, bfloat16 or float16 (got code %d)", (int)dtype);
      return TTHRML_ERR_ARG;
  }
}

extern "C" int tthrml_widen_i8(const int8_t* values, int64_t n, void* out, void* stream) {
  using namespace tthrml;
  if (n == 0) return TTHRML_OK;
  if (!values || !out || n < 0 || (uintptr_t)values % 16 || (uintptr_t)out % 16) {
    set_error("tthrml_widen_i8: buffers must be given and 16-byte aligned (got %lld elements)", (long long)n);
    return TTHRML_ERR_ARG;
  }
  const int64_t blocks = (n + 4095) / 4096;
  k_widen<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, (cudaStream_t)stream>>>(values, (__nv_bfloat16*)out, n);
  return launch_status("k_widen launch");
}
