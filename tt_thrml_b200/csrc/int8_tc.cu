// 8-bit integer product on the tensor cores (tcgen05.mma kind::i8, int32 accumulators):
//     y[m][n] = (sum_k q[m][k] w[n][k]) * (s_x[m] * s_w[n]) + bias[n],
// rows m (tokens / chains) and units n (channels) with one float32 scale each.  The sum is exact in int32 for
// K <= 131071 (2^31 / 128^2), so neither the split of K nor the order of the partial sums changes the result.
//
// k_int8_tile: one 128 x BN output tile per CTA cluster of S CTAs, each summing a contiguous share of the 128-wide K
// blocks.  Warp 0 loads (TMA, 128-byte swizzle, columns and rows behind the ends read as zeros), warp 1 multiplies,
// then all eight warps move the accumulator to shared memory, and CTA r of the cluster adds the S partial tiles of
// rows r, r + S, ... over distributed shared memory, scales and stores them as whole rows.
#include "int8_common.cuh"
#include "tc_common.cuh"

namespace tthrml {
namespace {

constexpr int kTileThreads = 256;

struct ProductArgs {
  const float* x_scale;  // [M]; NULL: ones
  const float* w_scale;  // [N]
  const float* bias;     // [N] or NULL
  void* out;             // [M][out_ld]
  int64_t out_ld;
  int32_t out_dtype;
  int32_t vector_store;  // rows of `out` are aligned for stores of four elements
  int32_t M, N;
  int32_t num_k;         // 128-column blocks of K
  int32_t box_m;         // rows per A load (16, 32, 64 or 128)
  int* error;
};

template <int BN>
struct TileShape {
  static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int kPitch = BN + 4;  // words per row of the staged accumulator: rows start four banks apart
  static constexpr int kSmem = 1024 + kStages * kStage + 256;
  static_assert(128 * kPitch * 4 <= kStages * kStage, "the staged tile reuses the operand stages");
};

// Instruction descriptor: D int32, A and B signed 8-bit, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}
__device__ __forceinline__ int4 ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// Four consecutive values of a row from column n (n % 4 == 0).
__device__ __forceinline__ void store4(const ProductArgs& a, int64_t m, int n, const float (&y)[4]) {
  const int64_t at = m * a.out_ld + n;
  if (a.vector_store && n + 4 <= a.N) {
    if (a.out_dtype == TTHRML_DT_F32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
    } else if (a.out_dtype == TTHRML_DT_BF16) {
      __nv_bfloat162 p[2] = {__floats2bfloat162_rn(y[0], y[1]), __floats2bfloat162_rn(y[2], y[3])};
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at) = *reinterpret_cast<uint2*>(p);
    } else {
      __half2 p[2] = {__floats2half2_rn(y[0], y[1]), __floats2half2_rn(y[2], y[3])};
      *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(a.out) + at) = *reinterpret_cast<uint2*>(p);
    }
    return;
  }
  for (int i = 0; i < 4 && n + i < a.N; ++i) {
    if (a.out_dtype == TTHRML_DT_F32)
      reinterpret_cast<float*>(a.out)[at + i] = y[i];
    else if (a.out_dtype == TTHRML_DT_BF16)
      reinterpret_cast<__nv_bfloat16*>(a.out)[at + i] = __float2bfloat16_rn(y[i]);
    else
      reinterpret_cast<__half*>(a.out)[at + i] = __float2half_rn(y[i]);
  }
}

template <int BN>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_int8_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, ProductArgs a) {
  using S = TileShape<BN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S::kStages * S::kStage);
  uint64_t* empty = full + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int n_blocks = (a.N + BN - 1) / BN;
  const int tile = (int)(blockIdx.x / split);
  const int m0 = (tile / n_blocks) * 128, n0 = (tile % n_blocks) * BN;
  const int k_first = (int)((int64_t)a.num_k * rank / split), k_last = (int)((int64_t)a.num_k * (rank + 1) / split);

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"((uint32_t)BN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t bytes = (uint32_t)(a.box_m * 128 + S::kBBytes);
      int issued = 0;
      for (int kb = k_first; kb < k_last; ++kb, ++issued) {
        const int s = issued % S::kStages;
        if (!mbar_wait(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
          atomicExch(a.error, kErrEmptyWait);
          break;
        }
        mbar_expect_tx(&full[s], bytes);
        unsigned char* t = tiles + s * S::kStage;
        tma_load_2d(t, &map_a, &full[s], kb * 128, m0);
        tma_load_2d(t + S::kABytes, &map_b, &full[s], kb * 128, n0);
      }
      // the copies issued must land before the stages are used again or the CTA exits
      for (int j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
        if (!mbar_wait(&full[j % S::kStages], (uint32_t)(j / S::kStages) & 1u)) atomicExch(a.error, kErrFullWait);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int used = 0;
      for (int kb = k_first; kb < k_last; ++kb, ++used) {
        const int s = used % S::kStages;
        if (!mbar_wait(&full[s], (uint32_t)(used / S::kStages) & 1u)) {
          atomicExch(a.error, kErrFullWait);
          break;
        }
        tc_fence_after();
        const unsigned char* t = tiles + s * S::kStage;
        const uint64_t ad = umma_desc_sw128(t), bd = umma_desc_sw128(t + S::kABytes);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)  // K = 32 bytes per MMA
          umma_i8(tmem, ad + 2ull * kk, bd + 2ull * kk, idesc_i8(128, BN), (used > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      umma_commit(done);
    }
  }
  const bool ok = mbar_wait(done, 0u);
  if (!ok && lane == 0) atomicExch(a.error, kErrAccWait);
  tc_fence_after();
  __syncthreads();  // the stages are free: every copy has landed and every MMA has read them

  int32_t* staged = reinterpret_cast<int32_t*>(tiles);
  if (ok && m0 + (warp & 3) * 32 < a.M) {
    const int row = (warp & 3) * 32 + lane;
    for (int c = (warp >> 2) * 32; c < BN; c += 64) {
      float v[32];
      tmem_load32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
      int4* dst = reinterpret_cast<int4*>(staged + row * S::kPitch + c);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        dst[q] = make_int4(__float_as_int(v[4 * q]), __float_as_int(v[4 * q + 1]), __float_as_int(v[4 * q + 2]),
                           __float_as_int(v[4 * q + 3]));
    }
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)BN));
  }

  const int rows = min(128, a.M - m0);
  const int mine = (rows - rank + split - 1) / split;  // rows rank, rank + split, ...
  for (int i = threadIdx.x; i < mine * (BN / 4); i += kTileThreads) {
    const int row = rank + (i / (BN / 4)) * split, c = (i % (BN / 4)) * 4, n = n0 + c;
    if (n >= a.N) continue;
    int4 sum;
    if (split == 1) {
      sum = *reinterpret_cast<const int4*>(staged + row * S::kPitch + c);
    } else {
      const uint32_t at = smem_u32(staged + row * S::kPitch + c);
      sum = make_int4(0, 0, 0, 0);
      for (int r = 0; r < split; ++r) {
        const int4 p = ld_cluster(at, (uint32_t)r);
        sum.x += p.x;
        sum.y += p.y;
        sum.z += p.z;
        sum.w += p.w;
      }
    }
    const float sx = a.x_scale ? __ldg(a.x_scale + m0 + row) : 1.0f;
    const int32_t v[4] = {sum.x, sum.y, sum.z, sum.w};
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int nn = n + j < a.N ? n + j : a.N - 1;
      y[j] = __fmul_rn((float)v[j], __fmul_rn(sx, __ldg(a.w_scale + nn)));
      if (a.bias) y[j] = __fadd_rn(y[j], __ldg(a.bias + nn));
    }
    store4(a, m0 + row, n, y);
  }
  if (split > 1) cluster_sync_all();  // no CTA leaves while another still reads its shared memory
}

// Tensor map of an 8-bit matrix [rows][cols] with rows `pitch` bytes apart, read in (box_rows x 128) tiles, 128-byte swizzle.
int make_map_i8(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, uint32_t box_rows) {
  EncodeTiledFn fn;
  int rc = encode_fn(&fn);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128u, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for a %lld x %lld 8-bit matrix", (int)r, (long long)rows,
              (long long)cols);
    return TTHRML_ERR_CUDA;
  }
  return TTHRML_OK;
}

template <int BN>
int launch_tile(const CUtensorMap& ma, const CUtensorMap& mb, const ProductArgs& a, int split, cudaStream_t st) {
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  void* params[3] = {(void*)&ma, (void*)&mb, (void*)&a};
  return launch_clusters((const void*)k_int8_tile<BN>, (unsigned)(tiles * split), (unsigned)split, kTileThreads,
                         TileShape<BN>::kSmem, params, st, "k_int8_tile launch");
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_int8_product(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* weights,
                                   int64_t w_pitch, const float* w_scale, int64_t rows, int64_t units, int64_t cols,
                                   const float* bias, void* out, int32_t out_dtype, int64_t out_ld, int32_t* error,
                                   void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  if (!x || !weights || !w_scale || !out || !error) {
    set_error("tthrml_int8_product: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (rows < 1 || units < 1 || cols < 1 || cols > TTHRML_INT8_MAX_COLS || rows > 0x7fffff00LL || units > 0x7fffff00LL ||
      ((rows + 127) / 128) * ((units + 63) / 64) > 0x0fffffffLL) {
    set_error("tthrml_int8_product: sizes out of range (rows %lld, units %lld, columns %lld of at most %d)",
              (long long)rows, (long long)units, (long long)cols, TTHRML_INT8_MAX_COLS);
    return TTHRML_ERR_ARG;
  }
  if (out_dtype == TTHRML_DT_I8 || dtype_bytes(out_dtype) == 0) {
    set_error("tthrml_int8_product: output type must be float32, bfloat16 or float16 (got code %d)", (int)out_dtype);
    return TTHRML_ERR_ARG;
  }
  if ((uintptr_t)x % 16 || (uintptr_t)weights % 16 || x_pitch % 16 || w_pitch % 16 || x_pitch < cols ||
      w_pitch < cols || out_ld < units) {
    set_error("tthrml_int8_product: 8-bit operands must be 16-byte aligned with pitches >= cols that are multiples "
              "of 16, and output rows must not overlap (got pitches %lld, %lld, %lld)", (long long)x_pitch,
              (long long)w_pitch, (long long)out_ld);
    return TTHRML_ERR_ARG;
  }
  ProductArgs a;
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.bias = bias;
  a.out = out;
  a.out_ld = out_ld;
  a.out_dtype = out_dtype;
  const int64_t quad = 4 * dtype_bytes(out_dtype);
  a.vector_store = (uintptr_t)out % quad == 0 && out_ld % 4 == 0;
  a.M = (int32_t)rows;
  a.N = (int32_t)units;
  a.num_k = (int32_t)((cols + 127) / 128);
  a.box_m = rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 64 ? 64 : 128));
  a.error = error;
  CUtensorMap ma, mb;
  int rc = make_map_i8(&ma, x, rows, cols, x_pitch, (uint32_t)a.box_m);
  if (rc) return rc;
  const int bn = 128;
  rc = make_map_i8(&mb, weights, units, cols, w_pitch, (uint32_t)bn);
  if (rc) return rc;
  return launch_tile<128>(ma, mb, a, 1, (cudaStream_t)stream);
}
