// 8-bit integer product on the tensor cores (tcgen05.mma kind::i8, int32 accumulators):
//     y[m][n] = (sum_k q[m][k] w[n][k]) * (s_x[m] * s_w[n]) + bias[n],
// rows m (tokens / chains) and units n (channels) with one float32 scale each.  The sum is exact in int32 for
// K <= 131071 (2^31 / 128^2), so neither the split of K nor the order of the partial sums changes the result.
//
// k_int8_tile: one 128 x BN output tile per CTA cluster of S CTAs, each summing a contiguous share of the 128-wide K
// blocks.  Warp 0 loads (TMA, 128-byte swizzle, columns and rows behind the ends read as zeros), warp 1 multiplies,
// then all eight warps move the accumulator to shared memory, and CTA r of the cluster adds the S partial tiles of
// rows r, r + S, ... over distributed shared memory, scales and stores them as whole rows.
//
// k_int8_pair: persistent clusters of two CTAs walk 256 x 256 tiles (tcgen05 cta_group::2, as the bf16 kernel of the dense
// sweeps does): each CTA holds 128 rows of either operand per stage, the even CTA issues every MMA, two TMEM accumulators let
// the epilogue of one tile run under the main loop of the next.  The epilogue stores the scaled sums, or takes them as
// the fields of a dense block and draws its new state.
#include "dense_draw.cuh"
#include "int8_common.cuh"

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
  int32_t vector_store;  // tiles: rows of `out` are aligned for stores of four elements; pairs: bytes they are aligned to
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
  static constexpr int kSmem = 1024 + kStages * kStage + 256 /*barriers*/ + 512 /*row scales*/;
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
  float* row_scale_of = reinterpret_cast<float*>(tiles + S::kStages * S::kStage + 256);

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
  // the scales and biases of the four columns that this thread will store, and the rows' scales
  constexpr int kGroups = BN / 4, kRowStep = kTileThreads / kGroups;
  const int c0 = ((int)threadIdx.x % kGroups) * 4, n = n0 + c0;
  float sw[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool live = n + j < a.N;
    sw[j] = live ? __ldg(a.w_scale + n + j) : 0.0f;
    bias[j] = live && a.bias ? __ldg(a.bias + n + j) : 0.0f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    const bool one = elect_one();
    const uint32_t bytes = (uint32_t)(a.box_m * 128 + S::kBBytes);
    const int ahead = min(S::kStages, k_last - k_first);
    for (int s = 0; s < ahead; ++s) {  // the weights of the first stages, while the rows are still being quantised
      if (one) {
        mbar_expect_tx(&full[s], bytes);
        tma_load_2d(tiles + s * S::kStage + S::kABytes, &map_b, &full[s], (k_first + s) * 128, n0);
      }
    }
    wait_for_previous_kernel();
    for (int s = 0; s < ahead; ++s)
      if (one) tma_load_2d(tiles + s * S::kStage, &map_a, &full[s], (k_first + s) * 128, m0);
    int issued = ahead;
    for (int kb = k_first + ahead; kb < k_last; ++kb, ++issued) {
      const int s = issued % S::kStages;
      if (!mbar_wait_all(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
        if (one) atomicExch(a.error, kErrEmptyWait);
        break;
      }
      if (one) {
        mbar_expect_tx(&full[s], bytes);
        unsigned char* t = tiles + s * S::kStage;
        tma_load_2d(t, &map_a, &full[s], kb * 128, m0);
        tma_load_2d(t + S::kABytes, &map_b, &full[s], kb * 128, n0);
      }
      __syncwarp();
    }
    // the copies issued must land before the stages are used again or the CTA exits
    for (int j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&full[j % S::kStages], (uint32_t)(j / S::kStages) & 1u) && one) atomicExch(a.error, kErrFullWait);
  } else if (warp == 1) {
    const bool one = elect_one();
    int used = 0;
    for (int kb = k_first; kb < k_last; ++kb, ++used) {
      const int s = used % S::kStages;
      if (!mbar_wait_all(&full[s], (uint32_t)(used / S::kStages) & 1u)) {
        if (one) atomicExch(a.error, kErrFullWait);
        break;
      }
      tc_fence_after();
      const unsigned char* t = tiles + s * S::kStage;
      const uint64_t ad = umma_desc_sw128(t), bd = umma_desc_sw128(t + S::kABytes);
      if (one) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)  // K = 32 bytes per MMA
          umma_i8(tmem, ad + 2ull * kk, bd + 2ull * kk, idesc_i8(128, BN), (used > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (one) umma_commit(done);
    __syncwarp();
  } else if (warp >= 4) {
    const int row = (int)threadIdx.x - 128;
    wait_for_previous_kernel();
    row_scale_of[row] = a.x_scale && m0 + row < a.M ? a.x_scale[m0 + row] : 1.0f;
  }
  const bool ok = mbar_wait_warp(done, 0u);
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
  if (n < a.N) {
#pragma unroll 4
    for (int row = rank + (int)threadIdx.x / kGroups * split; row < rows; row += kRowStep * split) {
      int4 sum;
      if (split == 1) {
        sum = *reinterpret_cast<const int4*>(staged + row * S::kPitch + c0);
      } else {
        const uint32_t at = smem_u32(staged + row * S::kPitch + c0);
        int4 p[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < split) p[r] = ld_cluster(at, (uint32_t)r);
        sum = p[0];
#pragma unroll
        for (int r = 1; r < 8; ++r)
          if (r < split) sum.x += p[r].x, sum.y += p[r].y, sum.z += p[r].z, sum.w += p[r].w;
      }
      const float sx = row_scale_of[row];
      const int32_t v[4] = {sum.x, sum.y, sum.z, sum.w};
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = __fmul_rn((float)v[j], __fmul_rn(sx, sw[j]));
        if (a.bias) y[j] = __fadd_rn(y[j], bias[j]);
      }
      store4(a, m0 + row, n, y);
    }
  }
  if (split > 1) cluster_sync_all();  // no CTA leaves while another still reads its shared memory
}

// ---------------------------------------------------------------------------
// CTA-pair kernel
// ---------------------------------------------------------------------------
constexpr int kPairStages = 6, kPairStage = 2 * 128 * 128, kPairThreads = 320, kPairWarps = 8;
constexpr int kScaleWords = 2 * 512;  // scales and biases of a tile's units, two tiles
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + 256 + kScaleWords * 4 + kPairWarps * 32 * kTurnPitch;
enum : int { kStoreFields = 0, kDrawSpins = 1, kDrawGaussians = 2 };

struct PairArgs {
  ProductArgs p;
  DenseArgs d;       // draws: bias, variates, counters; M, N
  int8_t* spins;     // [M][N] new spins
  __nv_bfloat16* values;  // [M][N] new gaussian values
};

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc_i8(256, 256)), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u),
      "r"(0u), "r"(0u), "r"(0u));
}

// Sums of 32 consecutive units of one row, scaled: (float)sum * (s_x * s_w); sw: the units' scales in shared memory.
__device__ __forceinline__ void scale_chunk(float sx, const float* sw, float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 w = reinterpret_cast<const float4*>(sw)[q];
    v[4 * q] = __fmul_rn((float)__float_as_int(v[4 * q]), __fmul_rn(sx, w.x));
    v[4 * q + 1] = __fmul_rn((float)__float_as_int(v[4 * q + 1]), __fmul_rn(sx, w.y));
    v[4 * q + 2] = __fmul_rn((float)__float_as_int(v[4 * q + 2]), __fmul_rn(sx, w.z));
    v[4 * q + 3] = __fmul_rn((float)__float_as_int(v[4 * q + 3]), __fmul_rn(sx, w.w));
  }
}

// Adds the biases to one 32-column chunk of 32 rows (lane = row m) and stores it.
__device__ __forceinline__ void store_chunk(const ProductArgs& a, int m, int n_first, const float* bias, float (&y)[32],
                                            unsigned char* turn) {
  if (a.bias) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 b = reinterpret_cast<const float4*>(bias)[q];
      y[4 * q] = __fadd_rn(y[4 * q], b.x);
      y[4 * q + 1] = __fadd_rn(y[4 * q + 1], b.y);
      y[4 * q + 2] = __fadd_rn(y[4 * q + 2], b.z);
      y[4 * q + 3] = __fadd_rn(y[4 * q + 3], b.w);
    }
  }
  unsigned char* out = reinterpret_cast<unsigned char*>(a.out);
  const int m0 = m - (int)(threadIdx.x & 31), live = min(32, a.N - n_first);
  if (a.out_dtype == TTHRML_DT_F32) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = make_uint4(__float_as_uint(y[16 * half + 4 * q]), __float_as_uint(y[16 * half + 4 * q + 1]),
                          __float_as_uint(y[16 * half + 4 * q + 2]), __float_as_uint(y[16 * half + 4 * q + 3]));
      const int left = min(16, live - 16 * half);
      if (left > 0) store_rows<4>(w, turn, out, a.out_ld * 4, 4 * (int64_t)(n_first + 16 * half), m0, a.M, 4 * left, a.vector_store);
    }
    return;
  }
  uint4 w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = y[8 * q + 2 * j], hi = y[8 * q + 2 * j + 1];
      if (a.out_dtype == TTHRML_DT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    w[q] = make_uint4(p[0], p[1], p[2], p[3]);
  }
  store_rows<4>(w, turn, out, a.out_ld * 2, 2 * (int64_t)n_first, m0, a.M, 2 * live, a.vector_store);
}

template <int EPI, bool VARIATES>
__global__ void __launch_bounds__(kPairThreads, 1)
    k_int8_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ PairArgs args) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + kPairStages * kPairStage);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* unit_scales = reinterpret_cast<float*>(tiles + kPairStages * kPairStage + 256);  // [2][scales 256, biases 256]
  unsigned char* turns = reinterpret_cast<unsigned char*>(unit_scales + kScaleWords);

  const ProductArgs& a = args.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int m_blocks = (a.M + 255) / 256, n_blocks = (a.N + 255) / 256;
  const int n_tiles = m_blocks * n_blocks;
  const int first = (int)cluster_id_x(), step = (int)n_clusters_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kPairWarps);  // every epilogue warp of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  int last_it[2] = {-1, -1};

  if (warp == 0) {  // producer (both CTAs): this CTA's halves of the A and B slices
    const bool one = elect_one();
    int64_t issued = 0;
    bool failed = false;
    for (int t = first; t < n_tiles && !failed; t += step) {
      int mb, nb;
      tile_coords(t, m_blocks, n_blocks, args.d.group, mb, nb);
      for (int kb = 0; kb < a.num_k; ++kb) {
        const int s = (int)(issued % kPairStages);
        if (!mbar_wait_all(&empty[s], ((uint32_t)(issued / kPairStages) & 1u) ^ 1u)) {
          if (one) atomicExch(a.error, kErrEmptyWait);
          failed = true;
          break;
        }
        if (one) {
          if (leader) mbar_expect_tx(&full[s], 2 * kPairStage);  // the stage's bytes of both CTAs
          unsigned char* st = tiles + s * kPairStage;
          const uint32_t bar = smem_u32(&full[s]) & kPeerMask;
          tma_load_2d_pair(st, &map_a, bar, kb * 128, mb * 256 + (int)rank * 128);
          tma_load_2d_pair(st + kPairStage / 2, &map_b, bar, kb * 128, nb * 256 + (int)rank * 128);
        }
        __syncwarp();
        ++issued;
      }
    }
    // every stage this CTA filled has been consumed (released by the leader's MMAs) before exit
    for (int64_t j = issued > kPairStages ? issued - kPairStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&empty[j % kPairStages], (uint32_t)(j / kPairStages) & 1u) && one) atomicExch(a.error, kErrEmptyWait);
  } else if (warp == 1) {
    if (leader) {  // MMA issue: the leader only
      const bool one = elect_one();
      int64_t used = 0;
      int it = 0;
      bool failed = false;
      for (int t = first; t < n_tiles && !failed; t += step, ++it) {
        const int b = it & 1;
        if (!mbar_wait_all(&acc_empty[b], ((uint32_t)(it >> 1) & 1u) ^ 1u)) {
          if (one) atomicExch(a.error, kErrAccWait);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(b * 256);
        for (int kb = 0; kb < a.num_k; ++kb) {
          const int s = (int)(used % kPairStages);
          if (!mbar_wait_all(&full[s], (uint32_t)(used / kPairStages) & 1u)) {
            if (one) atomicExch(a.error, kErrFullWait);
            failed = true;
            break;
          }
          tc_fence_after();
          const unsigned char* st = tiles + s * kPairStage;
          const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + kPairStage / 2);
          if (one) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // K = 32 bytes per MMA
              umma_i8_pair(d, ad + 2ull * kk, bd + 2ull * kk, (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[s]);  // the stage is free again in both CTAs
          }
          __syncwarp();
          ++used;
        }
        if (one) umma_commit_pair(&acc_full[b]);  // both CTAs' accumulator halves complete
        __syncwarp();
        last_it[b] = it;
      }
    }
  } else {
    const int quad = warp & 3, grp = (warp - 2) >> 2;
    unsigned char* turn = turns + (warp - 2) * 32 * kTurnPitch;
    int it = 0;
    bool failed = false;
    for (int t = first; t < n_tiles; t += step, ++it) {
      int mb, nb;
      tile_coords(t, m_blocks, n_blocks, args.d.group, mb, nb);
      const int b = it & 1;
      const int m = mb * 256 + (int)rank * 128 + quad * 32 + lane;
      const float sx = a.x_scale && m < a.M ? __ldg(a.x_scale + m) : 1.0f;
      // the tile's scales and biases, a unit per thread; two buffers, so that a warp may run one tile ahead
      float* sw = unit_scales + b * 512;
      {
        const int j = (int)threadIdx.x - 64, n = nb * 256 + j;
        sw[j] = n < a.N ? __ldg(a.w_scale + n) : 0.0f;
        sw[256 + j] = EPI == kStoreFields && a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (!failed && !mbar_wait_all(&acc_full[b], (uint32_t)(it >> 1) & 1u)) {
        if (lane == 0) atomicExch(a.error, kErrAccWait);
        failed = true;
      }
      if (failed) continue;  // on to the next tile's barrier, which the other warps wait at
      tc_fence_after();
      const uint32_t sweep = args.d.sweep + (EPI != kStoreFields && args.d.ctl ? args.d.ctl->sweep : 0u);
      const uint64_t sd = EPI != kStoreFields && args.d.ctl ? args.d.ctl->seed : args.d.seed;
      const PhiloxKeys keys = philox_keys(seed_lo(sd), seed_hi(sd));
      const float inv = 1.0f / __fadd_rn(args.d.precision, 1e-6f);
      const float sd_g = sqrtf(inv);
      const int64_t vs = VARIATES ? (int64_t)(sweep % (uint32_t)(args.d.variates_sweeps > 0 ? args.d.variates_sweeps : 1)) : 0;
      for (int c = grp; c < 8 && nb * 256 + c * 32 < a.N; c += 2) {
        const int n_first = nb * 256 + c * 32;
        float v[32];
        tmem_load32(tmem + (uint32_t)(b * 256) + ((uint32_t)(quad * 32) << 16) + (uint32_t)(c * 32), v);
        scale_chunk(sx, sw + c * 32, v);
        if (EPI == kStoreFields) {
          store_chunk(a, m, n_first, sw + 256 + c * 32, v, turn);
        } else if (EPI == kDrawSpins) {  // N is a multiple of 32; lanes behind the last chain draw for it and store nothing
          uint32_t near;
          const uint32_t down = spin_chunk<VARIATES>(args.d, v, m < a.M ? m : a.M - 1, n_first, sweep, keys, vs, near);
          uint32_t w[8];  // four spins a word: bit -> 0x01 / 0xFF
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t four = (down >> (4 * q)) & 15u;
            w[q] = 0x01010101u | (((four * 0x00204081u) & 0x01010101u) * 0xFEu);
          }
          const uint4 row[2] = {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
          store_rows<2>(row, turn, reinterpret_cast<unsigned char*>(args.spins), a.N, n_first, m - lane, a.M, 32, 16);
        } else {
          float f[32];
          gauss_chunk<VARIATES>(args.d, v, m < a.M ? m : a.M - 1, n_first, sweep, keys, inv, sd_g, vs, f);
          uint4 row[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(f[8 * q + 2 * j], f[8 * q + 2 * j + 1]);
              p[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            row[q] = make_uint4(p[0], p[1], p[2], p[3]);
          }
          store_rows<4>(row, turn, reinterpret_cast<unsigned char*>(args.values), 2 * (int64_t)a.N, 2 * (int64_t)n_first,
                        m - lane, a.M, 64, 16);
        }
        __syncwarp();  // the next TMEM load is a warp's
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&acc_empty[b]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1 && leader) {
    // every MMA the pair issued has completed (in both CTAs' TMEM) before TMEM is freed
    if (lane == 0) {
      for (int b = 0; b < 2; ++b)
        if (last_it[b] >= 0) (void)mbar_wait(&acc_full[b], (uint32_t)(last_it[b] >> 1) & 1u);
    }
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA frees TMEM or exits while the other may still signal it
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
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

// Clusters of 1, 2, 4 and 8 CTAs of k_int8_tile<BN> that are resident at once on the current device.
template <int BN>
int resident_tiles(const int** out) {
  static std::mutex mu;
  static int known[64][4] = {};
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= 64) return cuda_status(e == cudaSuccess ? cudaErrorInvalidDevice : e, "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < 4 && !known[dev][3]; ++i) {
    ClusterFit fit;
    const int rc = cluster_fit((const void*)k_int8_tile<BN>, 1u << i, kTileThreads, TileShape<BN>::kSmem, &fit);
    if (rc) return rc;
    known[dev][i] = fit.clusters;
  }
  *out = known[dev];
  return TTHRML_OK;
}

// Estimated clocks of the tiles on clusters of S CTAs: per wave the blocks of a CTA's share of K (block_clocks), at least 360
// clocks each to issue, the tile's store, and for S > 1 a barrier and the partial tiles.  The constants are those with which the choice among
// (BN, S) and the pair kernel came out best over 56 sizes of 3 to 8192 rows with every choice measured: 1.5 % behind the
// fastest on average, 28 % at most.  256 x 8192 x 4096: (256, 4) 15.7 us of 15.7 to 76; 256 x 4096 x 8192: (128, 1) 14.6 of
// 14.6 to 109; 64 x 5008 x 2048: (64, 4) 8.1 of 8.1 to 24.
template <int BN>
int consider(const ProductArgs& a, int64_t& best, int& bn, int& split) {
  const int* resident;
  const int rc = resident_tiles<BN>(&resident);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  for (int i = 0; i < 4 && (1 << i) <= a.num_k; ++i) {
    const int s = 1 << i;
    const int64_t waves = (tiles + resident[i] - 1) / resident[i];
    const int64_t block = block_clocks((a.box_m + BN) * 128, (tiles < resident[i] ? tiles : resident[i]) * s, std::max(2 * BN, 360));
    const int64_t c = 8300 + waves * ((a.num_k + s - 1) / s * block + 20 * BN +
                                      (s > 1 ? 850 + (int64_t)(a.M < 128 ? a.M : 128) * BN / 10 : 0));
    if (c < best) best = c, bn = BN, split = s;
  }
  return TTHRML_OK;
}

template <int BN>
int launch_tile(const int8_t* weights, int64_t cols, int64_t w_pitch, const CUtensorMap& ma, const ProductArgs& a,
                int split, bool early, cudaStream_t st) {
  CUtensorMap mb;
  const int rc = make_map_i8(&mb, weights, a.N, cols, w_pitch, (uint32_t)BN);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  void* params[3] = {(void*)&ma, (void*)&mb, (void*)&a};
  return launch_clusters((const void*)k_int8_tile<BN>, (unsigned)(tiles * split), (unsigned)split, kTileThreads,
                         TileShape<BN>::kSmem, params, st, "k_int8_tile launch", early);
}

// As many clusters as are resident at once walk the tiles.
int launch_pair(const void* fn, const CUtensorMap& ma, const CUtensorMap& mb, PairArgs& a, int64_t cols, cudaStream_t st) {
  ClusterFit fit;
  const int rc = cluster_fit(fn, 2, kPairThreads, kPairSmem, &fit);
  if (rc) return rc;
  const int64_t mblk = (a.p.M + 255) / 256, tiles = mblk * ((a.p.N + 255) / 256);
  const int64_t g = ((int64_t)32 << 20) / (256 * cols);  // raster groups of about 32 MiB of A panels, as in the bf16 kernel
  a.d.group = (int32_t)(g < 1 ? 1 : (g > mblk ? mblk : g));
  const int64_t clusters = tiles < fit.clusters ? tiles : fit.clusters;
  void* params[3] = {(void*)&ma, (void*)&mb, (void*)&a};
  return launch_clusters(fn, (unsigned)(2 * clusters), 2, kPairThreads, kPairSmem, params, st,
                         "k_int8_pair launch");
}

}  // namespace
}  // namespace tthrml

namespace {

// early: the rows were quantised by the kernel just before on the stream, which this one need not wait for at once
int int8_product(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* weights, int64_t w_pitch,
                 const float* w_scale, int64_t rows, int64_t units, int64_t cols, const float* bias, void* out,
                 int32_t out_dtype, int64_t out_ld, int32_t* error, bool early, void* stream) {
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
  cudaStream_t st = (cudaStream_t)stream;
  CUtensorMap ma, mb;
  int rc;
  const void* pair_fn = (const void*)k_int8_pair<kStoreFields, false>;
  ClusterFit fit;
  rc = cluster_fit(pair_fn, 2, kPairThreads, kPairSmem, &fit);
  if (rc) return rc;
  int64_t best = INT64_MAX;
  int bn = 128, split = 1;
  if ((rc = consider<64>(a, best, bn, split)) || (rc = consider<128>(a, best, bn, split)) ||
      (rc = consider<256>(a, best, bn, split)))
    return rc;
  // the pair kernel overlaps a tile's epilogue with the next tile's loop
  const int64_t pairs = ((rows + 255) / 256) * ((units + 255) / 256), at_once = pairs < fit.clusters ? pairs : fit.clusters;
  if ((pairs + fit.clusters - 1) / fit.clusters * a.num_k * block_clocks(kPairStage, 2 * at_once, 684) + 13700 < best) {
    rc = make_map_i8(&ma, x, rows, cols, x_pitch, 128u);
    if (rc == TTHRML_OK) rc = make_map_i8(&mb, weights, units, cols, w_pitch, 128u);
    if (rc) return rc;
    PairArgs pa = {};
    pa.p = a;
    const uint64_t alignment = (uint64_t)(uintptr_t)out | (uint64_t)(out_ld * dtype_bytes(out_dtype));  // of the rows
    pa.p.vector_store = alignment % 16 == 0 ? 16 : (alignment % 8 == 0 ? 8 : (alignment % 4 == 0 ? 4 : 0));
    return launch_pair(pair_fn, ma, mb, pa, cols, st);
  }
  rc = make_map_i8(&ma, x, rows, cols, x_pitch, (uint32_t)a.box_m);
  if (rc) return rc;
  if (bn == 64) return launch_tile<64>(weights, cols, w_pitch, ma, a, split, early, st);
  if (bn == 128) return launch_tile<128>(weights, cols, w_pitch, ma, a, split, early, st);
  return launch_tile<256>(weights, cols, w_pitch, ma, a, split, early, st);
}

}  // namespace

extern "C" int tthrml_int8_product(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* weights,
                                   int64_t w_pitch, const float* w_scale, int64_t rows, int64_t units, int64_t cols,
                                   const float* bias, void* out, int32_t out_dtype, int64_t out_ld, int32_t* error,
                                   void* stream) {
  return int8_product(x, x_pitch, x_scale, weights, w_pitch, w_scale, rows, units, cols, bias, out, out_dtype, out_ld,
                      error, false, stream);
}

extern "C" int tthrml_int8_field_sample(const int8_t* source, int64_t source_pitch, const float* source_scale,
                                        const int8_t* weights_nk, int64_t w_pitch, const float* w_scale,
                                        int64_t n_chains, int64_t n_units, int64_t n_sources, const float* bias,
                                        int32_t family, float precision, void* out_state, int64_t row0,
                                        int64_t chain_offset, const float* variates, int64_t variates_sweeps,
                                        uint64_t seed, uint32_t sweep, const tthrml_run_ctl* ctl, int32_t* error,
                                        void* stream) {
  using namespace tthrml;
  if (!source || !weights_nk || !w_scale || !out_state || !error) {
    set_error("tthrml_int8_field_sample: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (n_chains <= 0 || n_units <= 0 || n_units % 32 || n_sources <= 0 || n_sources > TTHRML_INT8_MAX_COLS ||
      n_chains > 0x7fffff00LL || n_units > 0x7fffff00LL || ((n_chains + 255) / 256) * ((n_units + 255) / 256) > 0x0fffffffLL) {
    set_error("tthrml_int8_field_sample: units must be a multiple of 32 and sources at most %d (got %lld chains, %lld "
              "units, %lld sources)", TTHRML_INT8_MAX_COLS, (long long)n_chains, (long long)n_units, (long long)n_sources);
    return TTHRML_ERR_ARG;
  }
  if (family != TTHRML_SPIN && family != TTHRML_GAUSSIAN) {
    set_error("tthrml_int8_field_sample: family must be spin or gaussian");
    return TTHRML_ERR_ARG;
  }
  if (chain_offset % 4 || (uintptr_t)source % 16 || (uintptr_t)weights_nk % 16 || source_pitch % 16 || w_pitch % 16 ||
      source_pitch < n_sources || w_pitch < n_sources || (uintptr_t)out_state % 16 || (bias && (uintptr_t)bias % 16)) {
    set_error("tthrml_int8_field_sample: buffers must be 16-byte aligned, pitches multiples of 16 not below the sources "
              "and chain_offset a multiple of 4 (got pitches %lld, %lld)", (long long)source_pitch, (long long)w_pitch);
    return TTHRML_ERR_ARG;
  }
  PairArgs pa = {};
  pa.p.x_scale = source_scale;
  pa.p.w_scale = w_scale;
  pa.p.M = (int32_t)n_chains;
  pa.p.N = (int32_t)n_units;
  pa.p.num_k = (int32_t)((n_sources + 127) / 128);
  pa.p.error = error;
  pa.d.bias = bias;
  pa.d.variates = variates;
  pa.d.variates_sweeps = variates_sweeps;
  pa.d.M = n_chains;
  pa.d.N = n_units;
  pa.d.K = n_sources;
  pa.d.row0 = row0;
  pa.d.chain_offset = chain_offset;
  pa.d.seed = seed;
  pa.d.sweep = sweep;
  pa.d.family = family;
  pa.d.precision = precision;
  pa.d.ctl = ctl;
  pa.spins = (int8_t*)out_state;
  pa.values = (__nv_bfloat16*)out_state;
  CUtensorMap ma, mb;
  int rc = make_map_i8(&ma, source, n_chains, n_sources, source_pitch, 128u);
  if (rc == TTHRML_OK) rc = make_map_i8(&mb, weights_nk, n_units, n_sources, w_pitch, 128u);
  if (rc) return rc;
  const void* fn = family == TTHRML_SPIN ? (variates ? (const void*)k_int8_pair<kDrawSpins, true>
                                                     : (const void*)k_int8_pair<kDrawSpins, false>)
                                         : (variates ? (const void*)k_int8_pair<kDrawGaussians, true>
                                                     : (const void*)k_int8_pair<kDrawGaussians, false>);
  return launch_pair(fn, ma, mb, pa, n_sources, (cudaStream_t)stream);
}

extern "C" int tthrml_int8_linear(const void* x, int32_t x_dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                  int64_t col_stride, void* workspace, int64_t workspace_bytes, const int8_t* weights,
                                  int64_t w_pitch, const float* w_scale, int64_t units, const float* bias, void* out,
                                  int32_t out_dtype, int64_t out_ld, int32_t* error, void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  if (rows < 0 || cols < 1 || cols > TTHRML_INT8_MAX_COLS) {
    set_error("tthrml_int8_linear: sizes out of range (rows %lld, columns %lld of at most %d)", (long long)rows,
              (long long)cols, TTHRML_INT8_MAX_COLS);
    return TTHRML_ERR_ARG;
  }
  if (tthrml_int8_linear_workspace(rows, cols) == 0 && col_stride == 1 && (rows == 1 || row_stride >= cols))
    return tthrml_int8_product_few(x, x_dtype, row_stride, nullptr, weights, w_pitch, w_scale, rows, units, cols, bias,
                                   out, out_dtype, out_ld, stream);
  const int64_t pitch = (cols + 15) / 16 * 16, need = rows * pitch + (rows * 4 + 15) / 16 * 16;
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need) {
    set_error("tthrml_int8_linear: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
              (long long)workspace_bytes);
    return TTHRML_ERR_ARG;
  }
  int8_t* q = (int8_t*)workspace;
  float* scale = (float*)(q + rows * pitch);
  const int rc = tthrml_quantize_rows(x, x_dtype, rows, cols, row_stride, col_stride, q, pitch, scale, stream);
  if (rc) return rc;
  return int8_product(q, pitch, scale, weights, w_pitch, w_scale, rows, units, cols, bias, out, out_dtype, out_ld, error,
                      true, stream);
}

extern "C" int64_t tthrml_int8_linear_workspace(int64_t rows, int64_t cols) {
  const int64_t pitch = (cols + 15) / 16 * 16, wide = rows <= 1 ? 1 : 2;
  if (rows <= 2 && wide * pitch <= TTHRML_INT8_FEW_BYTES) return 0;
  return rows * pitch + (rows * 4 + 15) / 16 * 16;
}
