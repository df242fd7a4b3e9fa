// Rows to 4-bit floating point values with their scales (formula and layout: fp4_common.cuh), and back to float32.
//
// k_fp4_quantize<T, W>: one pass, W warps per row, as few as hold it in registers (1024 elements a warp, at most eight
// warps; longer rows read their tail again), as the 8-bit quantisation does.  A lane holds eight columns at a time, two
// lanes a block: its maximum is one shuffle away.  Bound: memory (b bytes read and 9/16 written per element), close to the
// instructions (72 % of the issue slots): 8192 x 4096 bfloat16 in 20.5 us (4.2 TB/s), float32 in 24.7 (6.2).
#include "fp4_common.cuh"

namespace tthrml {
namespace {

struct Fp4Out {
  unsigned char* codes;
  int64_t pitch;  // bytes
  unsigned char* blocks;
  float* scale;
};

template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(256, 4)
    k_fp4_quantize(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int contiguous, Fp4Out o) {
  __shared__ uint32_t part[8];
  let_next_kernel_start();
  wait_for_previous_kernel();
  constexpr int kKept = 4, kStep = 32 * W * 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (int)threadIdx.x & (32 * W - 1);
  const int64_t row = (int64_t)blockIdx.x * (8 / W) + warp / W;  // up to the end of the last 128 rows
  const bool live = row < rows;
  const int end = (int)fp4_up(cols, 256), code_cols = live ? (int)(2 * o.pitch) : 0;
  const T* xr = x + (live ? row : 0) * rs;
  const uint32_t off = (uint32_t)((uintptr_t)xr & 15u);
  const RowReader<T, ALIGNED> in = {xr, live ? (int32_t)cols : 0, cs, contiguous ? (off ? kShifted : kAligned) : kElements, off};
  Vec8<T> kept[kKept];
  float most[kKept];  // of each vector
  float all = 0.0f;
  const auto largest = [](const Vec8<T>& v) {
    MaxOf<T> m;
    add_vector<T>(m, v);
    return m.value();
  };
#pragma unroll
  for (int v = 0; v < kKept; ++v) kept[v] = in.vector(v * kStep + 8 * t);
#pragma unroll
  for (int v = 0; v < kKept; ++v) {
    most[v] = largest(kept[v]);
    all = max_abs(all, most[v]);
  }
  for (int c = kKept * kStep + 8 * t; c < in.cols; c += kStep) all = max_abs(all, largest(in.vector(c)));
  uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(all));
  if (W > 1) {
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, part[warp / W * W + i]);
  }
  const Fp4RowScale s = fp4_row_scale(top);
  if (live && t == 0) o.scale[row] = s.scale;
  const float quotients = fp4_quotients(s.inv);
  unsigned char* codes = o.codes + row * o.pitch;
  unsigned char* blocks = o.blocks + fp4_scale_at(row, 0, end / 256);  // 512 bytes further per 64 columns
  const auto store = [&](const Vec8<T>& v, float mine, int c) {  // whole warps: c runs to a multiple of 256
    const uint32_t block = fp4_block_scale(max_abs(mine, __shfl_xor_sync(0xffffffffu, mine, 1)), s.inv);
    const float factor = fp4_code_factor(block, quotients);
    if ((lane & 1) == 0) blocks[c / 64 * 512 + (c / 16 & 3)] = (unsigned char)block;
    if (c >= code_cols) return;
    float f[8];
    unpack8(v, f);
    *reinterpret_cast<uint32_t*>(codes + c / 2) = fp4_codes8(f, factor);
  };
#pragma unroll
  for (int v = 0; v < kKept; ++v) {
    const int c = v * kStep + 8 * t;
    if (c - 8 * lane < end) store(kept[v], most[v], c);
  }
  for (int c = kKept * kStep + 8 * t; c - 8 * lane < end; c += kStep) {
    const Vec8<T> v = in.vector(c);
    store(v, largest(v), c);
  }
}

// The float32 values: (code * block) * scale, code * block exact.  A thread takes four columns at a time, so that a warp's
// store is 512 bytes in a row, of four rows whose loads go out together (8192 x 4096: eight columns a thread 42 us, four 34,
// of four rows 29).
constexpr int kValueRows = 4;
__global__ void __launch_bounds__(256) k_fp4_values(Fp4Out q, int64_t rows, int64_t cols, int vectors, float* __restrict__ out) {
  wait_for_previous_kernel();
  const int64_t r0 = (int64_t)blockIdx.x * kValueRows, c = (int64_t)blockIdx.y * 1024 + 4 * threadIdx.x;
  if (c >= cols) return;
  const int64_t k_blocks = fp4_up(cols, 256) / 256;
  uint32_t w[kValueRows], block[kValueRows];
  float scale[kValueRows];
#pragma unroll
  for (int i = 0; i < kValueRows; ++i) {
    const int64_t r = r0 + i < rows ? r0 + i : rows - 1;
    w[i] = __ldg(reinterpret_cast<const uint16_t*>(q.codes + r * q.pitch + c / 2));
    block[i] = __ldg(q.blocks + fp4_scale_at(r, c, k_blocks) + ((c >> 4) & 3));
    scale[i] = __ldg(q.scale + r);
  }
#pragma unroll
  for (int i = 0; i < kValueRows; ++i) {
    if (r0 + i >= rows) break;
    const float b = fp4_block_value(block[i]);
    const float2 lo = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)w[i], __NV_E2M1)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(w[i] >> 8), __NV_E2M1)));
    const float f[4] = {__fmul_rn(lo.x * b, scale[i]), __fmul_rn(lo.y * b, scale[i]), __fmul_rn(hi.x * b, scale[i]),
                        __fmul_rn(hi.y * b, scale[i])};
    float* o = out + (r0 + i) * cols + c;
    if (vectors) {
      *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) o[j] = f[j];
    }
  }
}

template <typename T>
int launch_quantize(const T* x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, const Fp4Out& o, cudaStream_t st) {
  const int contiguous = cs == 1;
  const bool aligned = contiguous && (uintptr_t)x % 16 == 0 && (rs * (int64_t)sizeof(T)) % 16 == 0;
  const int warps = cols <= 1024 ? 1 : (cols <= 2048 ? 2 : (cols <= 4096 ? 4 : 8));
  const unsigned grid = (unsigned)(fp4_up(rows, 128) / (8 / warps));
  const auto run = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(x, rows, cols, rs, cs, contiguous, o); };
  if (warps == 1)
    aligned ? run(k_fp4_quantize<T, 1, true>) : run(k_fp4_quantize<T, 1, false>);
  else if (warps == 2)
    aligned ? run(k_fp4_quantize<T, 2, true>) : run(k_fp4_quantize<T, 2, false>);
  else if (warps == 4)
    aligned ? run(k_fp4_quantize<T, 4, true>) : run(k_fp4_quantize<T, 4, false>);
  else
    aligned ? run(k_fp4_quantize<T, 8, true>) : run(k_fp4_quantize<T, 8, false>);
  return launch_status("k_fp4_quantize launch");
}

int check_rows(const char* what, const void* codes, int64_t pitch, const void* blocks, const float* scale, int64_t rows,
               int64_t cols) {
  if (!codes || !blocks || !scale) {
    set_error("%s: NULL argument", what);
    return TTHRML_ERR_ARG;
  }
  if (rows < 0 || cols < 1 || rows > 0x0fffffffLL || cols > TTHRML_FP4_MAX_COLS) {
    set_error("%s: sizes out of range (rows %lld, columns %lld of at most %d)", what, (long long)rows, (long long)cols,
              TTHRML_FP4_MAX_COLS);
    return TTHRML_ERR_ARG;
  }
  if (2 * pitch < cols || pitch % 16 || (uintptr_t)codes % 16 || (uintptr_t)blocks % 16) {
    set_error("%s: codes and block scales must be 16-byte aligned, codes with a pitch that is a multiple of 16 bytes and "
              "holds the columns (got pitch %lld for %lld columns)", what, (long long)pitch, (long long)cols);
    return TTHRML_ERR_ARG;
  }
  return TTHRML_OK;
}

}  // namespace
}  // namespace tthrml

extern "C" int64_t tthrml_fp4_scale_bytes(int64_t rows, int64_t cols) {
  return rows < 1 || cols < 1 ? 0 : tthrml::fp4_scale_bytes(rows, cols);
}

extern "C" int tthrml_fp4_quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                   int64_t col_stride, void* codes, int64_t pitch, void* blocks, float* scale, void* stream) {
  using namespace tthrml;
  if (rows == 0) return TTHRML_OK;
  const int rc = check_rows("tthrml_fp4_quantize", codes, pitch, blocks, scale, rows, cols);
  if (rc) return rc;
  if (!x || row_stride < 0 || col_stride < 1) {
    set_error("tthrml_fp4_quantize: NULL input or strides out of range (%lld, %lld)", (long long)row_stride,
              (long long)col_stride);
    return TTHRML_ERR_ARG;
  }
  const Fp4Out o = {(unsigned char*)codes, pitch, (unsigned char*)blocks, scale};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case TTHRML_DT_F32: return launch_quantize((const float*)x, rows, cols, row_stride, col_stride, o, st);
    case TTHRML_DT_BF16: return launch_quantize((const __nv_bfloat16*)x, rows, cols, row_stride, col_stride, o, st);
    case TTHRML_DT_F16: return launch_quantize((const __half*)x, rows, cols, row_stride, col_stride, o, st);
    default:
      set_error("tthrml_fp4_quantize: input type must be float32, bfloat16 or float16 (got code %d)", (int)dtype);
      return TTHRML_ERR_ARG;
  }
}

extern "C" int tthrml_fp4_values(const void* codes, int64_t pitch, const void* blocks, const float* scale, int64_t rows,
                                 int64_t cols, float* out, void* stream) {
  using namespace tthrml;
  if (rows == 0) return TTHRML_OK;
  const int rc = check_rows("tthrml_fp4_values", codes, pitch, blocks, scale, rows, cols);
  if (rc) return rc;
  if (!out || (uintptr_t)out % 16) {
    set_error("tthrml_fp4_values: the output must be given and 16-byte aligned");
    return TTHRML_ERR_ARG;
  }
  const Fp4Out q = {(unsigned char*)codes, pitch, (unsigned char*)blocks, (float*)scale};
  const dim3 grid((unsigned)((rows + kValueRows - 1) / kValueRows), (unsigned)((cols + 1023) / 1024));
  k_fp4_values<<<grid, 256, 0, (cudaStream_t)stream>>>(q, rows, cols, cols % 4 == 0, out);
  return launch_status("k_fp4_values launch");
}
