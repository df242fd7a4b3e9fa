// Product of a few rows (single tokens / chains) and 4-bit weights, the rows quantised in the same launch:
//     y[m][n] = (sum_k x[m][k] w[n][k]) * (s_x[m] * s_w[n]) + bias[n].
//
// Bound: the weights are read once (9/16 byte each).  Taking them apart on the CUDA cores costs more than that (conversions
// of codes to float16, or byte permutations and dp4a: 8192 x 4096 weights and one row in 14.0 and 11.4 us, 32768 x 4096 in 36 and
// 30), so the tensor cores multiply here too, with the roles changed: 128 units are the rows of the block-scaled MMA (operand
// A, loaded by TMA) and up to kFewRows rows of x its columns (operand B), which every CTA quantises itself into shared memory
// while its weights are on their way.
//
// A cluster of S CTAs takes 128 units, each CTA a contiguous share of the 256-wide blocks of K; the S partial sums are
// added over distributed shared memory in the order of the CTAs.
#include "fp4_tc.cuh"

namespace tthrml {
namespace {

constexpr int kFewThreads = 256, kFewStages = 4;
constexpr int kFewRows = 4, kColumns = 16;  // rows of x taken, and the MMA's columns that hold them
constexpr int kFewStage = 128 * 128 + kScales;          // codes and scales of 128 units and 256 columns
constexpr int kXBlock = kColumns * 128 + kScales;       // the same of x; the scales of rows behind the last are not used
constexpr int kFewMaxShare = 16;                        // blocks of K per CTA

struct Fp4FewArgs {
  const void* x;  // [M][x_ld], dense columns
  int64_t x_ld;
  const float* w_scale;
  const float* bias;
  void* out;
  int64_t out_ld;
  int32_t out_dtype, M, K, N, num_k;
  int* error;
};
__host__ __device__ constexpr int few_smem(int share) {
  return 1024 + kFewStages * kFewStage + share * kXBlock + kColumns * 128 * 4 /*sums*/ + 256 /*barriers*/;
}

template <typename T, int RP>
__global__ void __launch_bounds__(kFewThreads)
    k_fp4_few(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s, const Fp4FewArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int n0 = (int)(blockIdx.x / split) * 128;
  const int k_first = (int)((int64_t)a.num_k * rank / split), k_last = (int)((int64_t)a.num_k * (rank + 1) / split);
  const int share = k_last - k_first, most_share = (a.num_k + split - 1) / split;
  unsigned char* xs = stages + kFewStages * kFewStage;  // [share] codes of 16 rows, then their scales
  float* sums = reinterpret_cast<float*>(xs + most_share * kXBlock);  // [16][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(sums + kColumns * 128);
  uint64_t* empty = full + kFewStages;
  uint64_t* done = empty + kFewStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  __shared__ float row_scale[kFewRows];
  __shared__ uint32_t part[8];

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(64u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  const bool one = warp == 0 && elect_one();
  const auto load = [&](int i) {  // the i-th block of this CTA's share
    unsigned char* t = stages + i % kFewStages * kFewStage;
    uint64_t* bar = &full[i % kFewStages];
    mbar_expect_tx(bar, kFewStage);
    tma_load_2d(t, &map_w, bar, (k_first + i) * 128, n0);
    tma_load_2d(t + 128 * 128, &map_s, bar, 0, 2 * (n0 / 128 * a.num_k + k_first + i));
  };
  const int ahead = min(kFewStages, share);
  if (one) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < ahead; ++i) load(i);
  }
  __syncwarp();

  // 8 / RP warps per row: its largest magnitude, then the codes and scales of this CTA's columns
  {
    constexpr int kWarps = 8 / RP;
    const int m = warp / kWarps, w = warp % kWarps;
    const T* xr = reinterpret_cast<const T*>(a.x) + (int64_t)(m < a.M ? m : 0) * a.x_ld;
    const uint32_t off = (uint32_t)((uintptr_t)xr & 15u);
    const RowReader<T, false> in = {xr, m < a.M ? a.K : 0, 1, off ? kShifted : kAligned, off};
    float most[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 8 * lane + 256 * w; c < in.cols; c += 1024 * kWarps) {  // four vectors on their way at a time
      Vec8<T> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = in.vector(c + 256 * kWarps * u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        MaxOf<T> t;
        add_vector<T>(t, v[u]);
        most[u] = max_abs(most[u], t.value());
      }
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(max_abs(max_abs(most[0], most[1]), max_abs(most[2], most[3]))));
    if (kWarps > 1) {
      if (lane == 0) part[warp] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = max(top, part[warp / kWarps * kWarps + i]);
    }
    const Fp4RowScale s = fp4_row_scale(top);
    if (lane == 0 && w == 0) row_scale[m] = s.scale;
    const float quotients = fp4_quotients(s.inv);
#pragma unroll 2
    for (int i = w; i < share; i += kWarps) {
      const Vec8<T> v = in.vector((k_first + i) * 256 + 8 * lane);
      MaxOf<T> t;
      add_vector<T>(t, v);
      const float mine = t.value();
      const uint32_t block = fp4_block_scale(max_abs(mine, __shfl_xor_sync(0xffffffffu, mine, 1)), s.inv);
      float f[8];
      unpack8(v, f);
      const uint32_t codes = fp4_codes8(f, fp4_code_factor(block, quotients));
      unsigned char* b = xs + i * kXBlock;
      // the 128-byte swizzle: piece j of row r lies at j ^ (r & 7); the scales as the tensor core takes them
      *reinterpret_cast<uint32_t*>(b + m * 128 + 16 * ((lane >> 2) ^ (m & 7)) + 4 * (lane & 3)) = codes;
      if ((lane & 1) == 0) b[kColumns * 128 + (lane >> 3) * 512 + m * 16 + (lane >> 1 & 3)] = (unsigned char)block;
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads what was written here
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    int i = ahead;
    for (; i < share; ++i) {
      if (!mbar_wait_all(&empty[i % kFewStages], ((uint32_t)(i / kFewStages) & 1u) ^ 1u)) {
        if (one) atomicExch(a.error, kErrEmptyWait);
        break;
      }
      if (one) load(i);
      __syncwarp();
    }
    // the copies issued must land before the CTA exits
    for (int j = i > kFewStages ? i - kFewStages : 0; j < i; ++j)
      if (!mbar_wait_all(&full[j % kFewStages], (uint32_t)(j / kFewStages) & 1u) && one) atomicExch(a.error, kErrFullWait);
  } else if (warp == 1) {
    const bool issue = elect_one();
    const uint32_t w_scales = tmem + kColumns, x_scales = w_scales + 16;
    for (int i = 0; i < share; ++i) {
      const int s = i % kFewStages;
      if (!mbar_wait_all(&full[s], (uint32_t)(i / kFewStages) & 1u)) {
        if (issue) atomicExch(a.error, kErrFullWait);
        break;
      }
      tc_fence_after();
      const unsigned char *t = stages + s * kFewStage, *b = xs + i * kXBlock;
      const uint64_t ad = umma_desc_sw128(t), bd = umma_desc_sw128(b), sa = scales_desc(t + 128 * 128), sb = scales_desc(b + kColumns * 128);
      if (issue) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // 512 bytes of scales: 32 in the descriptor's units of 16
          copy_scales(w_scales + 4 * kk, sa + 32ull * kk);
          copy_scales(x_scales + 4 * kk, sb + 32ull * kk);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)  // K = 64 columns, 32 bytes, per MMA
          umma_fp4(tmem, ad + 2ull * kk, bd + 2ull * kk, idesc_fp4(128, kColumns), w_scales + 4 * kk, x_scales + 4 * kk,
                   (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (issue) umma_commit(done);
    __syncwarp();
  }
  const bool ok = mbar_wait_warp(done, 0u);
  if (!ok && lane == 0) atomicExch(a.error, kErrAccWait);
  tc_fence_after();
  if (warp < 4 && ok) {  // a unit per lane
    float v[16];
    tmem_load16(tmem + ((uint32_t)(warp * 32) << 16), v);
#pragma unroll
    for (int m = 0; m < kFewRows; ++m)
      if (m < a.M) sums[m * 128 + warp * 32 + lane] = v[m];
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(64u));
  }
  // CTA r of the cluster finishes its part of the units
  const int mine = 128 / split;
  for (int i = threadIdx.x; i < mine * a.M; i += kFewThreads) {
    const int m = i / mine, c = rank * mine + i % mine, n = n0 + c;
    if (n >= a.N) continue;
    float v = 0.0f;
    for (int r = 0; r < split; ++r) {
      uint32_t remote;
      float p;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(sums + m * 128 + c)), "r"(r));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(remote) : "memory");
      v = r ? v + p : p;
    }
    float y = __fmul_rn(v, __fmul_rn(row_scale[m], __ldg(a.w_scale + n)));
    if (a.bias) y = __fadd_rn(y, __ldg(a.bias + n));
    const int64_t at = (int64_t)m * a.out_ld + n;
    if (a.out_dtype == TTHRML_DT_F32)
      reinterpret_cast<float*>(a.out)[at] = y;
    else if (a.out_dtype == TTHRML_DT_BF16)
      reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    else
      reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(y);
  }
  if (split > 1) cluster_sync_all();  // no CTA leaves while another still reads its shared memory
}

template <typename T, int RP>
int launch_rows(const CUtensorMap& mw, const CUtensorMap& ms, const Fp4FewArgs& a, cudaStream_t st) {
  // the smallest split with which the CTAs fill the SMs and the rows fit, and no CTA without work
  const int tiles = (a.N + 127) / 128;
  int split = 1;
  while (split < 8 && 2 * split <= a.num_k && (tiles * split < 148 || (a.num_k + split - 1) / split > kFewMaxShare)) split *= 2;
  void* params[3] = {(void*)&mw, (void*)&ms, (void*)&a};
  return launch_clusters((const void*)k_fp4_few<T, RP>, (unsigned)(tiles * split), (unsigned)split, kFewThreads,
                         few_smem((a.num_k + split - 1) / split), params, st, "k_fp4_few launch");
}
template <typename T>
int launch(const CUtensorMap& mw, const CUtensorMap& ms, const Fp4FewArgs& a, cudaStream_t st) {
  if (a.M == 1) return launch_rows<T, 1>(mw, ms, a, st);
  return a.M == 2 ? launch_rows<T, 2>(mw, ms, a, st) : launch_rows<T, 4>(mw, ms, a, st);
}

}  // namespace
}  // namespace tthrml

// Whether tthrml_fp4_product_few takes the rows.  More rows, or more units than there are SMs for at once, are quicker
// quantised first (4096 columns; 1, 4 and 8 rows in 8.5, 9.9 and 11.6 us with 8192 units, where quantisation and tiles take
// 10.1; 32768 units in 21.3, 24.8 and 30 us against 18).
extern "C" int tthrml_fp4_few_rows(int64_t rows, int64_t cols, int64_t units) {
  return rows >= 1 && rows <= tthrml::kFewRows && cols >= 1 && cols <= 8 * tthrml::kFewMaxShare * 256 && units <= 148 * 128;
}

extern "C" int tthrml_fp4_product_few(const void* x, int32_t x_dtype, int64_t x_ld, const void* w_codes, int64_t w_pitch,
                                      const void* w_blocks, const float* w_scale, int64_t rows, int64_t units, int64_t cols,
                                      const float* bias, void* out, int32_t out_dtype, int64_t out_ld, int32_t* error, void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  if (!x || !w_codes || !w_blocks || !w_scale || !out || !error) {
    set_error("tthrml_fp4_product_few: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (!tthrml_fp4_few_rows(rows, cols, units) || units < 1) {
    set_error("tthrml_fp4_product_few: takes 1 to %d rows of up to %d columns and up to %d units (got %lld rows of %lld, %lld "
              "units)", kFewRows, 8 * kFewMaxShare * 256, 148 * 128, (long long)rows, (long long)cols, (long long)units);
    return TTHRML_ERR_ARG;
  }
  if (out_dtype == TTHRML_DT_I8 || dtype_bytes(out_dtype) == 0) {
    set_error("tthrml_fp4_product_few: output type must be float32, bfloat16 or float16 (got code %d)", (int)out_dtype);
    return TTHRML_ERR_ARG;
  }
  if ((uintptr_t)w_codes % 16 || (uintptr_t)w_blocks % 16 || w_pitch % 16 || 2 * w_pitch < cols || (rows > 1 && out_ld < units) ||
      x_ld < 0) {
    set_error("tthrml_fp4_product_few: codes and scales must be 16-byte aligned, codes with a pitch that is a multiple of 16 bytes "
              "and holds the columns, and output rows must not overlap (got pitches %lld, %lld)", (long long)w_pitch, (long long)out_ld);
    return TTHRML_ERR_ARG;
  }
  const Fp4FewArgs a = {x, x_ld, w_scale, bias, out, out_ld, out_dtype, (int32_t)rows, (int32_t)cols, (int32_t)units,
                        (int32_t)((cols + 255) / 256), error};
  CUtensorMap mw, ms;
  int rc = make_map_codes(&mw, w_codes, units, (cols + 1) / 2, w_pitch, 128u);
  if (rc == TTHRML_OK) rc = make_map_scales(&ms, w_blocks, units, cols);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  switch (x_dtype) {
    case TTHRML_DT_F32: return launch<float>(mw, ms, a, st);
    case TTHRML_DT_BF16: return launch<__nv_bfloat16>(mw, ms, a, st);
    case TTHRML_DT_F16: return launch<__half>(mw, ms, a, st);
    default:
      set_error("tthrml_fp4_product_few: input type must be float32, bfloat16 or float16 (got code %d)", (int)x_dtype);
      return TTHRML_ERR_ARG;
  }
}
