// Product of rows of 4-bit values on the tensor cores (tcgen05.mma kind::mxf4nvf4 with block scales):
//     y[m][n] = (sum_k x[m][k] w[n][k]) * (s_x[m] * s_w[n]) + bias[n],
// x and w codes times the scales of their blocks of 16 columns (fp4_common.cuh), the sums in float32.
//
// The codes of 256 columns are 128 bytes, a row of the 128-byte swizzle; their block scales (2048 bytes per 128 rows) go
// through shared memory into tensor memory (tcgen05.cp, replicated to the four quarters of the lanes), 4 columns per 128
// rows and 64 columns of K, right before the MMAs that use them: copies and MMAs of one thread run in order.
//
// k_fp4_tile: one 128 x BN output tile per CTA cluster of S CTAs, each summing a contiguous share of the 256-wide K
// blocks.  Warp 0 loads (TMA, columns and rows behind the ends read as zeros), warp 1 copies scales and multiplies, then all
// eight warps move the accumulator to shared memory, and CTA r of the cluster adds the S partial tiles of rows r, r + S, ...
// in the order of the CTAs, scales and stores them as whole rows.
//
// k_fp4_pair: persistent clusters of two CTAs walk 256 x 256 tiles (tcgen05 cta_group::2): an SM takes in at most 68 bytes a
// clock, and a 128 x 256 tile of one CTA needs 108 at the full MMA rate, a CTA of a pair 76 (16 KB of either operand, the
// scales of its rows and of all 256 units per 512 clocks).  The accumulator (256 columns) and the scales leave no room for a
// second one: the epilogue's eight warps take a finished tile into registers at once, free the accumulator for the next tile's
// MMAs and then scale and store.  8192 x 4096 x 8192 to bfloat16: 106 us (5.2 PFLOP/s, the tensor pipe 72 % active; the loads
// alone would leave it 71 to 76 %), in tiles of one CTA 205.
#include "fp4_tc.cuh"

namespace tthrml {
namespace {

constexpr int kTileThreads = 256;

struct Fp4Args {
  const float* x_scale;  // [M]
  const float* w_scale;  // [N]
  const float* bias;     // [N] or NULL
  void* out;             // [M][out_ld]
  int64_t out_ld;
  int32_t out_dtype;
  int32_t vector_store;  // rows of `out` are aligned for stores of four elements
  int32_t M, N;
  int32_t num_k;         // 256-column blocks of K
  int32_t box_m;         // rows per A load (16, 32, 64 or 128)
  int32_t group, align;  // pairs: raster, bytes that the rows of `out` are aligned to
  int32_t tma_store;     // `out` takes bulk tensor stores
  int* error;
};

template <int BN>
struct TileShape {
  static constexpr int kABytes = 128 * 128, kBBytes = BN * 128, kChunks = BN == 256 ? 2 : 1;  // row blocks of B's scales
  static constexpr int kStage = kABytes + kBBytes + kScales * (1 + kChunks);
  static constexpr int kStages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int kColumns = BN == 256 ? 512 : (BN == 128 ? 256 : 128);  // tensor memory: accumulator, scales of A, of B
  static constexpr int kPitch = BN + 4;  // words per row of the staged accumulator: rows start four banks apart
  static constexpr int kSmem = 1024 + kStages * kStage + 256 /*barriers*/ + 512 /*row scales*/;
  static_assert(128 * kPitch * 4 <= kStages * kStage, "the staged tile reuses the operand stages");
  static_assert(BN + 16 + 16 * kChunks <= kColumns, "accumulator and scales fit");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// Four consecutive values of a row from column n (n % 4 == 0).
__device__ __forceinline__ void store4(const Fp4Args& a, int64_t m, int n, const float (&y)[4]) {
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
    k_fp4_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb, Fp4Args a) {
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
                 "r"((uint32_t)S::kColumns));
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
    const uint32_t bytes = (uint32_t)(a.box_m * 128 + S::kBBytes + kScales * (1 + S::kChunks));
    const auto load_weights = [&](int s, int kb) {
      unsigned char* t = tiles + s * S::kStage;
      mbar_expect_tx(&full[s], bytes);
      tma_load_2d(t + S::kABytes, &map_b, &full[s], kb * 128, n0);
#pragma unroll
      for (int j = 0; j < S::kChunks; ++j)  // row blocks behind the last read as zeros
        tma_load_2d(t + S::kABytes + S::kBBytes + kScales * (1 + j), &map_sb, &full[s], 0, 2 * ((n0 / 128 + j) * a.num_k + kb));
    };
    const auto load_rows = [&](int s, int kb) {
      unsigned char* t = tiles + s * S::kStage;
      tma_load_2d(t, &map_a, &full[s], kb * 128, m0);
      tma_load_2d(t + S::kABytes + S::kBBytes, &map_sa, &full[s], 0, 2 * ((m0 / 128) * a.num_k + kb));
    };
    const int ahead = min(S::kStages, k_last - k_first);
    for (int s = 0; s < ahead; ++s)  // the weights of the first stages, while the rows are still being quantised
      if (one) load_weights(s, k_first + s);
    wait_for_previous_kernel();
    for (int s = 0; s < ahead; ++s)
      if (one) load_rows(s, k_first + s);
    int issued = ahead;
    for (int kb = k_first + ahead; kb < k_last; ++kb, ++issued) {
      const int s = issued % S::kStages;
      if (!mbar_wait_all(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
        if (one) atomicExch(a.error, kErrEmptyWait);
        break;
      }
      if (one) {
        load_weights(s, kb);
        load_rows(s, kb);
      }
      __syncwarp();
    }
    // the copies issued must land before the stages are used again or the CTA exits
    for (int j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&full[j % S::kStages], (uint32_t)(j / S::kStages) & 1u) && one) atomicExch(a.error, kErrFullWait);
  } else if (warp == 1) {
    const bool one = elect_one();
    const uint32_t a_scales = tmem + BN, b_scales = a_scales + 16;
    const uint32_t shift = BN == 64 && (n0 & 64) ? 2u : 0u;  // the tile's half of its 128 rows' scales
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
      const uint64_t sd = scales_desc(t + S::kABytes + S::kBBytes);
      if (one) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // 512 bytes of scales: 32 in the descriptor's units of 16
          copy_scales(a_scales + 4 * kk, sd + 32ull * kk);
#pragma unroll
          for (int j = 0; j < S::kChunks; ++j)
            copy_scales(b_scales + 4 * (S::kChunks * kk + j), sd + 128ull * (1 + j) + 32ull * kk);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)  // K = 64 columns, 32 bytes, per MMA
          umma_fp4(tmem, ad + 2ull * kk, bd + 2ull * kk, idesc_fp4(128, BN), a_scales + 4 * kk,
                   b_scales + 4 * S::kChunks * kk + shift, (used > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (one) umma_commit(done);
    __syncwarp();
  } else if (warp >= 4) {
    const int row = (int)threadIdx.x - 128;
    wait_for_previous_kernel();
    row_scale_of[row] = m0 + row < a.M ? a.x_scale[m0 + row] : 1.0f;
  }
  const bool ok = mbar_wait_warp(done, 0u);
  if (!ok && lane == 0) atomicExch(a.error, kErrAccWait);
  tc_fence_after();
  __syncthreads();  // the stages are free: every copy has landed and every MMA has read them

  float* staged = reinterpret_cast<float*>(tiles);
  if (ok && m0 + (warp & 3) * 32 < a.M) {
    const int row = (warp & 3) * 32 + lane;
    for (int c = (warp >> 2) * 32; c < BN; c += 64) {
      float v[32];
      tmem_load32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
      float4* dst = reinterpret_cast<float4*>(staged + row * S::kPitch + c);
#pragma unroll
      for (int q = 0; q < 8; ++q) dst[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::kColumns));
  }

  const int rows = min(128, a.M - m0);
  if (n < a.N) {
#pragma unroll 4
    for (int row = rank + (int)threadIdx.x / kGroups * split; row < rows; row += kRowStep * split) {
      float4 sum;
      if (split == 1) {
        sum = *reinterpret_cast<const float4*>(staged + row * S::kPitch + c0);
      } else {
        const uint32_t at = smem_u32(staged + row * S::kPitch + c0);
        float4 p[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < split) p[r] = ld_cluster_f4(at, (uint32_t)r);
        sum = p[0];
#pragma unroll
        for (int r = 1; r < 8; ++r)
          if (r < split) sum.x += p[r].x, sum.y += p[r].y, sum.z += p[r].z, sum.w += p[r].w;
      }
      const float sx = row_scale_of[row];
      const float v[4] = {sum.x, sum.y, sum.z, sum.w};
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = __fmul_rn(v[j], __fmul_rn(sx, sw[j]));
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
constexpr int kPairHalf = 128 * 128, kPairStage = 2 * kPairHalf + 3 * kScales, kPairStages = 5, kPairThreads = 320, kPairWarps = 8;
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + kPairWarps * kOutBytes + 256 +
                          512 * 4 /*scales and biases of a tile's units*/;
static_assert(32 * kTurnPitch <= kOutBytes, "unaligned outputs are turned in the same buffers");

__device__ __forceinline__ void umma_fp4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t a_scales,
                                              uint32_t b_scales, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc_fp4(256, 256)), "r"(a_scales), "r"(b_scales), "r"(accumulate));
}
// From each CTA's own shared memory into its own tensor memory.
__device__ __forceinline__ void copy_scales_pair(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc));
}
// Tile t -> (m, n) block: `group` row blocks at a time, row-fastest, so that the tiles in flight share panels in L2.
__device__ __forceinline__ void pair_tile(const Fp4Args& a, int t, int& mb, int& nb) {
  const int m_blocks = (a.M + 255) / 256, n_blocks = (a.N + 255) / 256;
  const int per = a.group * n_blocks, g = t / per, w = t - g * per;
  const int rows = min(a.group, m_blocks - g * a.group);
  mb = g * a.group + w % rows;
  nb = w / rows;
}

__global__ void __launch_bounds__(kPairThreads, 1)
    k_fp4_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
               const __grid_constant__ CUtensorMap map_out, const __grid_constant__ Fp4Args a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* turns = tiles + kPairStages * kPairStage;  // a buffer per warp
  uint64_t* full = reinterpret_cast<uint64_t*>(turns + kPairWarps * kOutBytes);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;
  uint64_t* acc_empty = acc_full + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 1);
  float* unit_scales = reinterpret_cast<float*>(turns + kPairWarps * kOutBytes + 256);  // scales 256, biases 256

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = ((a.M + 255) / 256) * ((a.N + 255) / 256);
  const int first = (int)cluster_id_x(), step = (int)n_clusters_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * kPairWarps);  // every epilogue warp of both CTAs
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
  wait_for_previous_kernel();
  int last_it = -1;

  if (warp == 0) {  // producer (both CTAs): this CTA's halves of the A and B slices, its rows' scales and all units'
    const bool one = elect_one();
    int64_t issued = 0;
    bool failed = false;
    for (int t = first; t < n_tiles && !failed; t += step) {
      int mb, nb;
      pair_tile(a, t, mb, nb);
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
          tma_load_2d_pair(st + kPairHalf, &map_b, bar, kb * 128, nb * 256 + (int)rank * 128);
          st += 2 * kPairHalf;  // row blocks behind the last read as zeros
          tma_load_2d_pair(st, &map_sa, bar, 0, 2 * ((mb * 2 + (int)rank) * a.num_k + kb));
          tma_load_2d_pair(st + kScales, &map_sb, bar, 0, 2 * (nb * 2 * a.num_k + kb));
          tma_load_2d_pair(st + 2 * kScales, &map_sb, bar, 0, 2 * ((nb * 2 + 1) * a.num_k + kb));
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
      const uint32_t a_scales = tmem + 256, b_scales = a_scales + 16;
      int64_t used = 0;
      int it = 0;
      bool failed = false;
      for (int t = first; t < n_tiles && !failed; t += step, ++it) {
        if (!mbar_wait_all(acc_empty, ((uint32_t)it & 1u) ^ 1u)) {
          if (one) atomicExch(a.error, kErrAccWait);
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < a.num_k; ++kb) {
          const int s = (int)(used % kPairStages);
          if (!mbar_wait_all(&full[s], (uint32_t)(used / kPairStages) & 1u)) {
            if (one) atomicExch(a.error, kErrFullWait);
            failed = true;
            break;
          }
          tc_fence_after();
          const unsigned char* st = tiles + s * kPairStage;
          const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + kPairHalf), sd = scales_desc(st + 2 * kPairHalf);
          if (one) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {  // 512 bytes of scales: 32 in the descriptor's units of 16
              copy_scales_pair(a_scales + 4 * kk, sd + 32ull * kk);
              copy_scales_pair(b_scales + 8 * kk, sd + 128ull + 32ull * kk);
              copy_scales_pair(b_scales + 8 * kk + 4, sd + 256ull + 32ull * kk);
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // K = 64 columns, 32 bytes, per MMA
              umma_fp4_pair(tmem, ad + 2ull * kk, bd + 2ull * kk, a_scales + 4 * kk, b_scales + 8 * kk,
                            (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[s]);  // the stage is free again in both CTAs
          }
          __syncwarp();
          ++used;
        }
        if (one) umma_commit_pair(acc_full);  // both CTAs' accumulator halves complete
        __syncwarp();
        last_it = it;
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    unsigned char* turn = turns + (warp - 2) * kOutBytes;
    const uint32_t buffer = smem_u32(turn);
    int it = 0;
    bool failed = false;
    // the scales and biases of a tile: its rows', a row per lane, and its units', a unit per thread; those of the next tile
    // are on their way while one is stored
    float next_x = 0.0f, next_w = 0.0f, next_b = 0.0f;
    const auto fetch = [&](int t) {
      int mb, nb;
      pair_tile(a, t, mb, nb);
      const int m = mb * 256 + (int)rank * 128 + quad * 32 + lane, n = nb * 256 + (int)threadIdx.x - 64;
      next_x = m < a.M ? __ldg(a.x_scale + m) : 0.0f;
      next_w = n < a.N ? __ldg(a.w_scale + n) : 0.0f;
      next_b = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
    };
    if (first < n_tiles) fetch(first);
    for (int t = first; t < n_tiles; t += step, ++it) {
      int mb, nb;
      pair_tile(a, t, mb, nb);
      const int m0 = mb * 256 + (int)rank * 128 + quad * 32;
      const float sx = next_x;
      float* sw = unit_scales;
      asm volatile("bar.sync 1, 256;" ::: "memory");  // every warp has read the scales of the tile before
      sw[(int)threadIdx.x - 64] = next_w;
      sw[(int)threadIdx.x + 192] = next_b;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (t + step < n_tiles) fetch(t + step);
      if (!failed && !mbar_wait_all(acc_full, (uint32_t)it & 1u)) {
        if (lane == 0) atomicExch(a.error, kErrAccWait);
        failed = true;
      }
      if (failed) continue;  // on to the next tile's barrier, which the other warps wait at
      tc_fence_after();
      float acc[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        tmem_load32_async(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128 + q * 32), acc[q]);
      tmem_wait(acc);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(acc_empty);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float* scales = sw + half * 128 + q * 32;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 w = reinterpret_cast<const float4*>(scales)[i];
          acc[q][4 * i] = __fmul_rn(acc[q][4 * i], __fmul_rn(sx, w.x));
          acc[q][4 * i + 1] = __fmul_rn(acc[q][4 * i + 1], __fmul_rn(sx, w.y));
          acc[q][4 * i + 2] = __fmul_rn(acc[q][4 * i + 2], __fmul_rn(sx, w.z));
          acc[q][4 * i + 3] = __fmul_rn(acc[q][4 * i + 3], __fmul_rn(sx, w.w));
        }
        if (a.bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 b = reinterpret_cast<const float4*>(scales + 256)[i];
            acc[q][4 * i] = __fadd_rn(acc[q][4 * i], b.x);
            acc[q][4 * i + 1] = __fadd_rn(acc[q][4 * i + 1], b.y);
            acc[q][4 * i + 2] = __fadd_rn(acc[q][4 * i + 2], b.z);
            acc[q][4 * i + 3] = __fadd_rn(acc[q][4 * i + 3], b.w);
          }
        }
      }
      const int n0 = nb * 256 + half * 128;
      if (a.tma_store) {
        if (m0 >= a.M) continue;
        const auto send = [&](const uint4 (&w)[8], int n) {
          if (n >= a.N) return;
          sent_rows_read<0>();
          stage_row(buffer, w);
          send_rows(&map_out, buffer, n, m0);
        };
        if (a.out_dtype == TTHRML_DT_F32) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[i] = make_uint4(__float_as_uint(acc[q][4 * i]), __float_as_uint(acc[q][4 * i + 1]),
                                __float_as_uint(acc[q][4 * i + 2]), __float_as_uint(acc[q][4 * i + 3]));
            send(w, n0 + q * 32);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            uint4 w[8];
            pack_row<4>(acc[q], a.out_dtype, w);
            pack_row<4>(acc[q + 1], a.out_dtype, w + 4);
            send(w, n0 + q * 32);
          }
        }
        continue;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + q * 32, live = min(32, a.N - n);
        if (live <= 0) break;
        store_values(acc[q], a.out_dtype, turn, (unsigned char*)a.out, a.out_ld, n, m0, a.M, live, a.align);
      }
    }
    sent_rows_done();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1 && leader) {
    // every MMA the pair issued has completed (in both CTAs' TMEM) before TMEM is freed
    if (lane == 0 && last_it >= 0) (void)mbar_wait(acc_full, (uint32_t)last_it & 1u);
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA frees TMEM or exits while the other may still signal it
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Clusters of 1, 2, 4 and 8 CTAs of k_fp4_tile<BN> that are resident at once on the current device.
template <int BN>
int resident_tiles(int (&out)[4]) {
  for (int i = 0; i < 4; ++i) {
    ClusterFit fit;
    const int rc = cluster_fit((const void*)k_fp4_tile<BN>, 1u << i, kTileThreads, TileShape<BN>::kSmem, &fit);
    if (rc) return rc;
    out[i] = fit.clusters;
  }
  return TTHRML_OK;
}

// Estimated clocks of the tiles on clusters of S CTAs, as for the 8-bit tiles: per wave the blocks of a CTA's share of K, the
// tile's store, and for S > 1 a barrier and the partial tiles.
template <int BN>
int consider(const Fp4Args& a, int64_t& best, int& bn, int& split) {
  int resident[4];
  const int rc = resident_tiles<BN>(resident);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  for (int i = 0; i < 4 && (1 << i) <= a.num_k; ++i) {
    const int s = 1 << i;
    const int64_t waves = (tiles + resident[i] - 1) / resident[i];
    const int64_t bytes = (a.box_m + BN) * 128 + kScales * (1 + TileShape<BN>::kChunks);
    const int64_t block = block_clocks(bytes, (tiles < resident[i] ? tiles : resident[i]) * s, std::max(2 * BN, 360));
    const int64_t c = 8300 + waves * ((a.num_k + s - 1) / s * block + 20 * BN +
                                      (s > 1 ? 850 + (int64_t)(a.M < 128 ? a.M : 128) * BN / 10 : 0));
    if (c < best) best = c, bn = BN, split = s;
  }
  return TTHRML_OK;
}

struct Fp4Operand {
  const void* codes;
  int64_t pitch;
  const void* blocks;
};

template <int BN>
int launch_tile(const Fp4Operand& w, int64_t cols, const CUtensorMap& ma, const CUtensorMap& msa, const CUtensorMap& msb,
                const Fp4Args& a, int split, bool early, cudaStream_t st) {
  CUtensorMap mb;
  const int rc = make_map_codes(&mb, w.codes, a.N, (cols + 1) / 2, w.pitch, (uint32_t)BN);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  void* params[5] = {(void*)&ma, (void*)&mb, (void*)&msa, (void*)&msb, (void*)&a};
  return launch_clusters((const void*)k_fp4_tile<BN>, (unsigned)(tiles * split), (unsigned)split, kTileThreads,
                         TileShape<BN>::kSmem, params, st, "k_fp4_tile launch", early);
}

}  // namespace
}  // namespace tthrml

namespace {

// early: the rows were quantised by the kernel just before on the stream, which this one need not wait for at once
int fp4_product(const void* x_codes, int64_t x_pitch, const void* x_blocks, const float* x_scale, const void* w_codes,
                int64_t w_pitch, const void* w_blocks, const float* w_scale, int64_t rows, int64_t units, int64_t cols,
                const float* bias, void* out, int32_t out_dtype, int64_t out_ld, int32_t* error, bool early, void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  if (!x_codes || !x_blocks || !x_scale || !w_codes || !w_blocks || !w_scale || !out || !error) {
    set_error("tthrml_fp4_product: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (rows < 1 || units < 1 || cols < 1 || cols > TTHRML_FP4_MAX_COLS || rows > 0x0fffffffLL || units > 0x0fffffffLL ||
      ((rows + 127) / 128) * ((units + 63) / 64) > 0x0fffffffLL ||
      std::max(fp4_scale_bytes(rows, cols), fp4_scale_bytes(units, cols)) / 1024 > 0x7fffff00LL) {
    set_error("tthrml_fp4_product: sizes out of range (rows %lld, units %lld, columns %lld of at most %d)", (long long)rows,
              (long long)units, (long long)cols, TTHRML_FP4_MAX_COLS);
    return TTHRML_ERR_ARG;
  }
  if (out_dtype == TTHRML_DT_I8 || dtype_bytes(out_dtype) == 0) {
    set_error("tthrml_fp4_product: output type must be float32, bfloat16 or float16 (got code %d)", (int)out_dtype);
    return TTHRML_ERR_ARG;
  }
  if ((uintptr_t)x_codes % 16 || (uintptr_t)w_codes % 16 || (uintptr_t)x_blocks % 16 || (uintptr_t)w_blocks % 16 ||
      x_pitch % 16 || w_pitch % 16 || 2 * x_pitch < cols || 2 * w_pitch < cols || out_ld < units) {
    set_error("tthrml_fp4_product: codes and scales must be 16-byte aligned, codes with pitches that are multiples of 16 bytes "
              "and hold the columns, and output rows must not overlap (got pitches %lld, %lld, %lld)", (long long)x_pitch,
              (long long)w_pitch, (long long)out_ld);
    return TTHRML_ERR_ARG;
  }
  Fp4Args a;
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.bias = bias;
  a.out = out;
  a.out_ld = out_ld;
  a.out_dtype = out_dtype;
  a.vector_store = (uintptr_t)out % (4 * dtype_bytes(out_dtype)) == 0 && out_ld % 4 == 0;
  a.M = (int32_t)rows;
  a.N = (int32_t)units;
  a.num_k = (int32_t)((cols + 255) / 256);
  a.box_m = rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 64 ? 64 : 128));
  a.error = error;
  cudaStream_t st = (cudaStream_t)stream;
  int64_t best = INT64_MAX;
  int bn = 128, split = 1, rc;
  if ((rc = consider<64>(a, best, bn, split)) || (rc = consider<128>(a, best, bn, split)) ||
      (rc = consider<256>(a, best, bn, split)))
    return rc;
  CUtensorMap ma, mb, msa, msb;
  // the pair kernel overlaps a tile's store with the next tile's loop
  ClusterFit fit;
  rc = cluster_fit((const void*)k_fp4_pair, 2, kPairThreads, kPairSmem, &fit);
  if (rc) return rc;
  const int64_t m_pairs = (rows + 255) / 256, pairs = m_pairs * ((units + 255) / 256);
  const int64_t at_once = pairs < fit.clusters ? pairs : fit.clusters;
  if ((pairs + fit.clusters - 1) / fit.clusters * (a.num_k * block_clocks(kPairStage, 2 * at_once, 512) + 1000) + 13700 < best) {
    rc = make_map_codes(&ma, x_codes, rows, (cols + 1) / 2, x_pitch, 128u);
    if (rc == TTHRML_OK) rc = make_map_codes(&mb, w_codes, units, (cols + 1) / 2, w_pitch, 128u);
    if (rc == TTHRML_OK) rc = make_map_scales(&msa, x_blocks, rows, cols);
    if (rc == TTHRML_OK) rc = make_map_scales(&msb, w_blocks, units, cols);
    if (rc) return rc;
    const uint64_t alignment = (uint64_t)(uintptr_t)out | (uint64_t)(out_ld * dtype_bytes(out_dtype));  // of the rows
    a.align = alignment % 16 == 0 ? 16 : (alignment % 8 == 0 ? 8 : (alignment % 4 == 0 ? 4 : 2));
    int64_t g = 1;  // about square rectangles of the tiles in flight
    while ((g + 1) * (g + 1) <= fit.clusters) ++g;
    a.group = (int32_t)(g < m_pairs ? g : m_pairs);
    CUtensorMap mo = ma;  // never used where the rows are not aligned
    // Bulk stores are the quicker way out, but take turns with the loads: 8192 x 8192 units in bfloat16, 1024, 2048 and 4096
    // columns, in 55, 68 and 114 us with them and 62, 71 and 107 us with stores from the warps.
    a.tma_store = a.num_k <= 8 && make_out_map(&mo, out, rows, units, out_ld, out_dtype);
    void* params[6] = {(void*)&ma, (void*)&mb, (void*)&msa, (void*)&msb, (void*)&mo, (void*)&a};
    return launch_clusters((const void*)k_fp4_pair, (unsigned)(2 * at_once), 2, kPairThreads, kPairSmem, params, st,
                           "k_fp4_pair launch", early);
  }
  rc = make_map_codes(&ma, x_codes, rows, (cols + 1) / 2, x_pitch, (uint32_t)a.box_m);
  if (rc == TTHRML_OK) rc = make_map_scales(&msa, x_blocks, rows, cols);
  if (rc == TTHRML_OK) rc = make_map_scales(&msb, w_blocks, units, cols);
  if (rc) return rc;
  const Fp4Operand w = {w_codes, w_pitch, w_blocks};
  if (bn == 64) return launch_tile<64>(w, cols, ma, msa, msb, a, split, early, st);
  if (bn == 128) return launch_tile<128>(w, cols, ma, msa, msb, a, split, early, st);
  return launch_tile<256>(w, cols, ma, msa, msb, a, split, early, st);
}

}  // namespace

extern "C" int tthrml_fp4_product(const void* x_codes, int64_t x_pitch, const void* x_blocks, const float* x_scale,
                                  const void* w_codes, int64_t w_pitch, const void* w_blocks, const float* w_scale,
                                  int64_t rows, int64_t units, int64_t cols, const float* bias, void* out, int32_t out_dtype,
                                  int64_t out_ld, int32_t* error, void* stream) {
  return fp4_product(x_codes, x_pitch, x_blocks, x_scale, w_codes, w_pitch, w_blocks, w_scale, rows, units, cols, bias, out,
                     out_dtype, out_ld, error, false, stream);
}

extern "C" int64_t tthrml_fp4_linear_workspace(int64_t rows, int64_t cols, int64_t units) {
  using namespace tthrml;
  if (rows < 1 || cols < 1 || rows > 0x0fffffffLL || cols > TTHRML_FP4_MAX_COLS || tthrml_fp4_few_rows(rows, cols, units)) return 0;
  return rows * (fp4_up(cols, 32) / 2) + fp4_scale_bytes(rows, cols) + fp4_up(rows * 4, 16);
}

extern "C" int tthrml_fp4_linear(const void* x, int32_t x_dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                 int64_t col_stride, void* workspace, int64_t workspace_bytes, const void* w_codes,
                                 int64_t w_pitch, const void* w_blocks, const float* w_scale, int64_t units, const float* bias,
                                 void* out, int32_t out_dtype, int64_t out_ld, int32_t* error, void* stream) {
  using namespace tthrml;
  if (rows == 0 || units == 0) return TTHRML_OK;
  const bool few = tthrml_fp4_few_rows(rows, cols, units) != 0;
  if (col_stride == 1 && few)
    return tthrml_fp4_product_few(x, x_dtype, row_stride, w_codes, w_pitch, w_blocks, w_scale, rows, units, cols, bias, out,
                                  out_dtype, out_ld, error, stream);
  const int64_t need = tthrml_fp4_linear_workspace(rows, cols, units);
  if (need == 0 && few) {
    set_error("tthrml_fp4_linear: few rows need dense columns (got a stride of %lld)", (long long)col_stride);
    return TTHRML_ERR_ARG;
  }
  if (need == 0) {
    set_error("tthrml_fp4_linear: sizes out of range (rows %lld, columns %lld of at most %d)", (long long)rows, (long long)cols,
              TTHRML_FP4_MAX_COLS);
    return TTHRML_ERR_ARG;
  }
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need) {
    set_error("tthrml_fp4_linear: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
              (long long)workspace_bytes);
    return TTHRML_ERR_ARG;
  }
  const int64_t pitch = fp4_up(cols, 32) / 2;
  unsigned char* codes = (unsigned char*)workspace;
  unsigned char* blocks = codes + rows * pitch;
  float* scale = (float*)(blocks + fp4_scale_bytes(rows, cols));
  const int rc = tthrml_fp4_quantize(x, x_dtype, rows, cols, row_stride, col_stride, codes, pitch, blocks, scale, stream);
  if (rc) return rc;
  return fp4_product(codes, pitch, blocks, scale, w_codes, w_pitch, w_blocks, w_scale, rows, units, cols, bias, out, out_dtype,
                     out_ld, error, true, stream);
}
