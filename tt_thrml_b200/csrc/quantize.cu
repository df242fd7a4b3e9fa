// Rows to 8-bit integers with one float32 scale per row (the formula stands in int8_common.cuh).
//
// One pass over the input: each row is read once, kept in registers while its largest magnitude is reduced, and
// written as packed bytes.  Bound: memory (b read + 1 written byte per element).
//   k_quantize_rows<T, W>: W warps per row (1 for rows up to 1024 elements, 8 above), eight consecutive elements
//     per thread and step; rows longer than the registers hold (W * 1024 elements) read their tail again.
//   k_quantize_cols<T>: rows whose consecutive elements are strided but whose neighbours are adjacent (a
//     transposed matrix): 32 rows per block, the lanes run along the rows, the bytes are transposed in shared memory.
#include "int8_common.cuh"

namespace tthrml {
namespace {

constexpr int kVecs = 4;  // vectors of eight elements that a thread keeps

template <typename T, int W>
__global__ void __launch_bounds__(256)
    k_quantize_rows(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int vectors,
                    int8_t* __restrict__ q, int64_t pitch, float* __restrict__ scale) {
  __shared__ uint32_t part[8];
  let_next_kernel_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = W == 1 ? lane : (int)threadIdx.x;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 8 + warp : (int64_t)blockIdx.x;
  if (row >= rows) return;  // W == 1: whole warps leave; W == 8: the grid has one block per row
  const T* xr = x + row * rs;
  constexpr int kStep = 32 * W * 8;  // elements per step of the group
  float kept[kVecs][8];
  uint32_t top = 0u;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int64_t c = (int64_t)v * kStep + 8 * t;
    if (vectors && c + 8 <= cols) {
      unpack8(load8(xr + c), kept[v]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) kept[v][i] = c + i < cols ? to_f32(xr[(c + i) * cs]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(kept[v][i]));
  }
  for (int64_t c = (int64_t)kVecs * kStep + 8 * t; c < cols; c += kStep) {
    if (vectors && c + 8 <= cols) {
      float f[8];
      unpack8(load8(xr + c), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, abs_bits(f[i]));
    } else {
      for (int i = 0; i < 8 && c + i < cols; ++i) top = max(top, abs_bits(to_f32(xr[(c + i) * cs])));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (W > 1) {
    if (lane == 0) part[warp] = top;
    __syncthreads();
    top = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) top = max(top, part[i]);
  }
  const RowScale s = row_scale(top);
  if (t == 0) scale[row] = s.scale;
  int8_t* qr = q + row * pitch;  // pitch is a multiple of 16; columns from cols to pitch are written as zeros
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int64_t c = (int64_t)v * kStep + 8 * t;
    if (c < pitch) {
      int32_t i8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) i8[i] = quantize(kept[v][i], s.inv);
      *reinterpret_cast<uint2*>(qr + c) = make_uint2(pack4(i8[0], i8[1], i8[2], i8[3]), pack4(i8[4], i8[5], i8[6], i8[7]));
    }
  }
  for (int64_t c = (int64_t)kVecs * kStep + 8 * t; c < pitch; c += kStep) {
    float f[8];
    if (vectors && c + 8 <= cols) {
      unpack8(load8(xr + c), f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i < cols ? to_f32(xr[(c + i) * cs]) : 0.0f;
    }
    int32_t i8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) i8[i] = quantize(f[i], s.inv);
    *reinterpret_cast<uint2*>(qr + c) = make_uint2(pack4(i8[0], i8[1], i8[2], i8[3]), pack4(i8[4], i8[5], i8[6], i8[7]));
  }
}

// Rows adjacent in memory (row stride 1): lane = row, warp w takes columns w, w + 8, ...
template <typename T>
__global__ void __launch_bounds__(256)
    k_quantize_cols(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t cs, int8_t* __restrict__ q,
                    int64_t pitch, float* __restrict__ scale) {
  __shared__ uint32_t part[8][32];
  __shared__ __align__(16) int8_t tile[32][144];  // 128 columns of 32 rows; the pitch spreads the rows over the banks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * 32, row = r0 + lane;
  const T* xr = x + row;
  uint32_t top = 0u;
  if (row < rows) {
#pragma unroll 8
    for (int64_t c = warp; c < cols; c += 8) top = max(top, abs_bits(to_f32(__ldg(xr + c * cs))));
  }
  part[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, part[i][lane]);
  const RowScale s = row_scale(top);
  if (warp == 0 && row < rows) scale[row] = s.scale;
  for (int64_t c0 = 0; c0 < pitch; c0 += 128) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t c = c0 + warp + 8 * i;
      const float v = row < rows && c < cols ? to_f32(__ldg(xr + c * cs)) : 0.0f;
      tile[lane][warp + 8 * i] = (int8_t)quantize(v, s.inv);
    }
    __syncthreads();
    const int r = threadIdx.x >> 3, b = (threadIdx.x & 7) * 16;  // 32 rows x 8 vectors of 16 bytes
    if (r0 + r < rows && c0 + b < pitch)
      *reinterpret_cast<uint4*>(q + (r0 + r) * pitch + c0 + b) = *reinterpret_cast<const uint4*>(&tile[r][b]);
    __syncthreads();
  }
}

template <typename T>
int launch_quantize(const T* x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int8_t* q, int64_t pitch,
                    float* scale, cudaStream_t st) {
  if (cs != 1 && rs == 1) {
    k_quantize_cols<T><<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(x, rows, cols, cs, q, pitch, scale);
    return launch_status("k_quantize_cols launch");
  }
  const int vectors = cs == 1 && (uintptr_t)x % 16 == 0 && (rs * (int64_t)sizeof(T)) % 16 == 0;
  if (cols <= 1024)
    k_quantize_rows<T, 1><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(x, rows, cols, rs, cs, vectors, q, pitch, scale);
  else
    k_quantize_rows<T, 8><<<(unsigned)rows, 256, 0, st>>>(x, rows, cols, rs, cs, vectors, q, pitch, scale);
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
  if (rows < 0 || cols < 1 || rows > 0x7fffffffLL || row_stride < 0 || col_stride < 1) {
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
