// Pair moments of two blocks over the chain batch, on the tensor cores (tcgen05.mma kind::f16):
//     out[i][j] (+)= sum_p s_p sum_c x_p[c][i] y_p[c][j],   with the unit sums sum_p s_p sum_c x_p[c][i] (and y).
// With a data phase (s = -1 / chains) and a model phase (s = 1 / chains) this is the gradient of a dense program's
// couplings and biases (the likelihood gradient of a Boltzmann machine; Ackley, Hinton and Sejnowski 1985).
//
// Both operands lie chain-major (the layout of the sampler's states), so the sum runs over the slow axis of each:
// the tiles are MN-major in shared memory (64 units x 64 chains per TMA box, 128-byte swizzle) and nothing is
// transposed.  Roles of a CTA's twelve warps:
//   warp 0      TMA loads into a ring of stages (chains and units behind the ends read as zeros);
//   warp 1      MMAs, kChunkBlocks blocks of 64 chains into one of two TMEM accumulators;
//   warps 2-9   add each finished accumulator, times its phase's scale, to float32 registers (half a tile row per thread);
//   warps 10-11 unit sums, a strip of 32 units at a time, beside the tiles.
// The tensor core's accumulation drops bits over long sums, so a sum longer than kChunkBlocks blocks is carried in registers
// with rounded float32 additions.
//
// k_pair_moments: for few tiles.  A cluster of S CTAs computes one 128 x BN tile, each CTA a contiguous share of the
// 64-chain blocks; the S partial tiles are added over distributed shared memory in the order of the ranks, so the result
// is the same every time.
// k_pair_moments_2sm: for many.  Persistent clusters of two CTAs walk 256 x 256 tiles (tcgen05 cta_group::2): an SM takes in
// at most 64 bytes a clock, and a 128 x 256 tile of one CTA needs 96 at the full MMA rate, a CTA of a pair 64.  The
// accumulating warps store a tile from their registers while the next one's first chunks are multiplied.
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace tthrml {
namespace {

constexpr int kMomentThreads = 384;
constexpr int kChunkBlocks = 16;  // 64-chain blocks per TMEM accumulation
constexpr int kSumUnits = 32;     // units per strip of unit sums

struct MomentMaps {
  CUtensorMap x[TTHRML_MAX_PHASES], y[TTHRML_MAX_PHASES];
};

struct MomentArgs {
  const void* x[TTHRML_MAX_PHASES];
  const void* y[TTHRML_MAX_PHASES];
  int64_t x_ld[TTHRML_MAX_PHASES], y_ld[TTHRML_MAX_PHASES];
  int64_t chains[TTHRML_MAX_PHASES];
  int32_t blocks[TTHRML_MAX_PHASES];  // 64-chain blocks
  float scale[TTHRML_MAX_PHASES], x_scale[TTHRML_MAX_PHASES], y_scale[TTHRML_MAX_PHASES];
  int32_t n_phases, total_blocks;
  int32_t M, N;
  float* out;
  int64_t out_ld;
  float* x_sum;
  float* y_sum;
  int32_t accumulate, vector_store;
  int32_t f16;         // elements are float16 (else bfloat16)
  int32_t tile_blocks;  // CTAs that compute tiles; any others sum units
  int32_t group;        // raster of the pair kernel
  int* error;
};

template <int BN>
struct MomentShape {
  static constexpr int kABytes = 128 * 64 * 2, kBBytes = BN * 64 * 2;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int kPitch = BN + 4;
  static constexpr int kSmem = 1024 + kStages * kStage + 256 /*barriers*/ + 256 /*unit sums*/;
  static_assert(128 * kPitch * 4 <= kStages * kStage, "the staged tile reuses the operand stages");
};

// D float32, A and B bfloat16 (or float16), both MN-major.
__device__ __forceinline__ uint32_t idesc_moments(int n, bool f16) {
  const uint32_t t = f16 ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
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

// The chunk that starts at block b of the concatenated phases: its phase, the block within it and its length (it ends
// with the phase, with the CTA's share or after kChunkBlocks blocks).
struct Chunk {
  int phase, block, length;
};
__device__ __forceinline__ Chunk chunk_at(const MomentArgs& a, int b, int last) {
  Chunk c;
  c.phase = 0;
  c.block = b;
  while (c.block >= a.blocks[c.phase]) c.block -= a.blocks[c.phase++];  // b < total: ends at a phase with blocks
  c.length = min(min(kChunkBlocks, a.blocks[c.phase] - c.block), last - b);
  return c;
}

__device__ __forceinline__ float elem(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(reinterpret_cast<const __half*>(p)[i])
             : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void add8(float (&s)[8], const uint4& w, bool f16) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (f16) {
      const __half2 h = *reinterpret_cast<const __half2*>(&v[i]);
      s[2 * i] += __low2float(h);
      s[2 * i + 1] += __high2float(h);
    } else {
      s[2 * i] += __uint_as_float(v[i] << 16);
      s[2 * i + 1] += __uint_as_float(v[i] & 0xFFFF0000u);
    }
  }
}

// Strip `strip` of the unit sums (32 units of x, then of y) by NT threads (t = 0 .. NT - 1, named barrier `bar`): four
// threads take the 64 bytes of a chain, NT / 4 chains at a time; the partial sums meet by shuffles and then in the order
// of the warps.  CLUSTER: the CTAs of a cluster take every `split`-th group of chains each, and rank 0 adds their sums in the
// order of the ranks.
template <int NT, bool CLUSTER>
__device__ __forceinline__ void unit_sums(const MomentArgs& a, int strip, int t, int bar, float* part, int rank, int split) {
  const int xs = a.x_sum ? (a.M + kSumUnits - 1) / kSumUnits : 0;
  const bool of_y = strip >= xs;
  const int u0 = (of_y ? strip - xs : strip) * kSumUnits, units = of_y ? a.N : a.M;
  const int u = u0 + (t & 3) * 8, lane = t >> 2;
  float total[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) total[i] = 0.0f;
  for (int p = 0; p < a.n_phases; ++p) {
    const char* base = reinterpret_cast<const char*>(of_y ? a.y[p] : a.x[p]);
    const int64_t ld = of_y ? a.y_ld[p] : a.x_ld[p];
    const float scale = of_y ? a.y_scale[p] : a.x_scale[p];
    if (scale == 0.0f && a.scale[p] != 0.0f) continue;  // a term of the products only; a phase of scale 0 is 0 times its sums
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.0f;
    if (u + 8 <= units) {  // rows start on 16 bytes and the units on multiples of eight
      const int64_t lanes = (int64_t)(NT / 4) * split, step = lanes * ld * 2;
      const int64_t first = (int64_t)(NT / 4) * rank + lane;
      const char* at = base + (first * ld + u) * 2;
      for (int64_t c = first; c < a.chains[p]; c += 16 * lanes, at += 16 * step) {  // 16 loads on their way at a time
        uint4 w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = c + i * lanes < a.chains[p] ? __ldg(reinterpret_cast<const uint4*>(at + i * step)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 16; ++i) add8(s, w[i], a.f16 != 0);
      }
    } else {
      for (int64_t c = (NT / 4) * rank + lane; c < a.chains[p]; c += (NT / 4) * split)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (u + i < units) s[i] += elem(base, c * ld + u + i, a.f16 != 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) total[i] = fmaf(scale, s[i], total[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) total[i] += __shfl_xor_sync(0xffffffffu, total[i], o);
  if ((t & 31) < 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[(t >> 5) * kSumUnits + (t & 3) * 8 + i] = total[i];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(NT) : "memory");
  float v = 0.0f;
  if (t < kSumUnits)
    for (int i = 0; i < NT / 32; ++i) v += part[i * kSumUnits + t];
  if (CLUSTER) {
    float* mine = part + NT / 32 * kSumUnits;
    if (t < kSumUnits) mine[t] = v;
    cluster_sync_all();
    if (rank == 0 && t < kSumUnits) {
      for (int r = 1; r < split; ++r) {
        uint32_t remote;
        float w;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine + t)), "r"(r));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(remote) : "memory");
        v += w;
      }
    }
    cluster_sync_all();  // before any CTA's next strip, or its end
  }
  if (rank == 0 && t < kSumUnits && u0 + t < units) {
    float* dst = (of_y ? a.y_sum : a.x_sum) + u0 + t;
    *dst = a.accumulate ? *dst + v : v;
  }
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(NT) : "memory");
}
__host__ __device__ inline int sum_strips(const MomentArgs& a) {
  return (a.x_sum ? (a.M + kSumUnits - 1) / kSumUnits : 0) + (a.y_sum ? (a.N + kSumUnits - 1) / kSumUnits : 0);
}
// The unit sums of CTAs that have no tile: a strip for a cluster where there are clusters enough, else for a CTA.
__device__ __forceinline__ void own_sums(const MomentArgs& a, float* part) {
  const int strips = sum_strips(a), others = (int)gridDim.x - a.tile_blocks, i = (int)blockIdx.x - a.tile_blocks;
  const int width = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  if (strips * width <= others) {
    if (i / width < strips) unit_sums<kMomentThreads, true>(a, i / width, (int)threadIdx.x, 1, part, rank, width);
  } else {
    for (int s = i; s < strips; s += others) unit_sums<kMomentThreads, false>(a, s, (int)threadIdx.x, 1, part, 0, 1);
  }
}
// The unit sums that fall to warps 10 and 11 of a tile's CTA.
__device__ __forceinline__ void side_sums(const MomentArgs& a, float* part) {
  if ((int)gridDim.x > a.tile_blocks) return;  // CTAs of their own sum the units
  const int strips = sum_strips(a);
  for (int s = blockIdx.x; s < strips; s += gridDim.x) unit_sums<64, false>(a, s, (int)threadIdx.x - 320, 1, part, 0, 1);
}

template <int BN>
__global__ void __launch_bounds__(kMomentThreads, 1)
    k_pair_moments(const __grid_constant__ MomentMaps maps, const __grid_constant__ MomentArgs a) {
  using S = MomentShape<BN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  if ((int)blockIdx.x >= a.tile_blocks) {  // whole clusters: the tile blocks are a multiple of the cluster size
    wait_for_previous_kernel();
    own_sums(a, reinterpret_cast<float*>(tiles));
    return;
  }
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S::kStages * S::kStage);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* side = reinterpret_cast<float*>(tiles + S::kStages * S::kStage + 256);  // [2][32]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int n_tiles = (a.N + BN - 1) / BN;
  const int tile = (int)(blockIdx.x / split);
  const int m0 = (tile / n_tiles) * 128, n0 = (tile % n_tiles) * BN;
  const int first = (int)((int64_t)a.total_blocks * rank / split), last = (int)((int64_t)a.total_blocks * (rank + 1) / split);

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"((uint32_t)(2 * BN)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);  // one arrival per accumulating warp
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  wait_for_previous_kernel();

  if (warp == 0) {
    const bool one = elect_one();
    int issued = 0;
    bool failed = false;
    for (int b = first; b < last && !failed;) {
      const Chunk c = chunk_at(a, b, last);
      for (int i = 0; i < c.length; ++i, ++issued) {
        const int s = issued % S::kStages;
        if (!mbar_wait_all(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
          if (one) atomicExch(a.error, kErrEmptyWait);
          failed = true;
          break;
        }
        if (one) {
          mbar_expect_tx(&full[s], S::kStage);
          unsigned char* t = tiles + s * S::kStage;
          const int chain = (c.block + i) * 64;
#pragma unroll
          for (int k = 0; k < 2; ++k) tma_load_2d(t + k * 8192, &maps.x[c.phase], &full[s], m0 + 64 * k, chain);
#pragma unroll
          for (int k = 0; k < BN / 64; ++k)
            tma_load_2d(t + S::kABytes + k * 8192, &maps.y[c.phase], &full[s], n0 + 64 * k, chain);
        }
        __syncwarp();
      }
      b += c.length;
    }
    // the copies issued must land before the stages are used again or the CTA exits
    for (int j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&full[j % S::kStages], (uint32_t)(j / S::kStages) & 1u) && one) atomicExch(a.error, kErrFullWait);
  } else if (warp == 1) {
    const bool one = elect_one();
    const uint32_t idesc = idesc_moments(BN, a.f16 != 0);
    int used = 0, chunk = 0;
    bool failed = false;
    for (int b = first; b < last && !failed; ++chunk) {
      const Chunk c = chunk_at(a, b, last);
      const int buf = chunk & 1;
      if (!mbar_wait_all(&acc_empty[buf], ((uint32_t)(chunk >> 1) & 1u) ^ 1u)) {
        if (one) atomicExch(a.error, kErrAccWait);
        failed = true;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + (uint32_t)(buf * BN);
      for (int i = 0; i < c.length; ++i, ++used) {
        const int s = used % S::kStages;
        if (!mbar_wait_all(&full[s], (uint32_t)(used / S::kStages) & 1u)) {
          if (one) atomicExch(a.error, kErrFullWait);
          failed = true;
          break;
        }
        tc_fence_after();
        const unsigned char* t = tiles + s * S::kStage;
        const uint64_t ad = umma_desc_mn128(t), bd = umma_desc_mn128(t + S::kABytes);
        if (one) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 chains per MMA: two groups of eight, 2048 bytes
            umma_f16(d, ad + 128ull * kk, bd + 128ull * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (one) umma_commit(&acc_full[buf]);
      __syncwarp();
      b += c.length;
    }
  } else if (warp >= 10) {
    side_sums(a, side);
  } else {
    // accumulating warps: lane = row within the warp's TMEM quadrant, half of the tile's columns each
    const int quad = warp & 3, half = (warp - 2) >> 2;
    float acc[BN / 2];
#pragma unroll
    for (int j = 0; j < BN / 2; ++j) acc[j] = 0.0f;
    int chunk = 0;
    for (int b = first; b < last; ++chunk) {
      const Chunk c = chunk_at(a, b, last);
      const int buf = chunk & 1;
      if (!mbar_wait_warp(&acc_full[buf], (uint32_t)(chunk >> 1) & 1u)) {
        if (lane == 0) atomicExch(a.error, kErrAccWait);
        break;
      }
      tc_fence_after();
      const float scale = a.scale[c.phase];
#pragma unroll
      for (int q = 0; q < BN / 64; ++q) {
        float v[32];
        tmem_load32(tmem + (uint32_t)(buf * BN + half * (BN / 2) + q * 32) + ((uint32_t)(quad * 32) << 16), v);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[q * 32 + j] = fmaf(scale, v[j], acc[q * 32 + j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&acc_empty[buf])) : "memory");
      b += c.length;
    }
    // Every MMA has read its stage: the last accumulator's barrier tracks all earlier ones.  The other warps may
    // still read their last accumulator, but no stage.
    float* staged = reinterpret_cast<float*>(tiles);
    float4* dst = reinterpret_cast<float4*>(staged + (quad * 32 + lane) * S::kPitch + half * (BN / 2));
#pragma unroll
    for (int j = 0; j < BN / 8; ++j) dst[j] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
  }
  tc_fence_before();
  __syncwarp();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN)));
  }

  const float* staged = reinterpret_cast<const float*>(tiles);
  const int rows = min(128, a.M - m0);
  const int mine = (rows - rank + split - 1) / split;  // rows rank, rank + split, ...
  for (int i = threadIdx.x; i < mine * (BN / 4); i += kMomentThreads) {
    const int row = rank + (i / (BN / 4)) * split, col = (i % (BN / 4)) * 4, n = n0 + col;
    if (n >= a.N) continue;
    float4 s;
    if (split == 1) {
      s = *reinterpret_cast<const float4*>(staged + row * S::kPitch + col);
    } else {
      const uint32_t at = smem_u32(staged + row * S::kPitch + col);
      s = ld_cluster_f4(at, 0u);
      for (int r = 1; r < split; ++r) {
        const float4 p = ld_cluster_f4(at, (uint32_t)r);
        s.x += p.x;
        s.y += p.y;
        s.z += p.z;
        s.w += p.w;
      }
    }
    float* o = a.out + (int64_t)(m0 + row) * a.out_ld + n;
    if (a.vector_store && n + 4 <= a.N) {
      if (a.accumulate) {
        const float4 old = *reinterpret_cast<const float4*>(o);
        s = make_float4(old.x + s.x, old.y + s.y, old.z + s.z, old.w + s.w);
      }
      *reinterpret_cast<float4*>(o) = s;
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
      for (int j = 0; j < 4 && n + j < a.N; ++j) o[j] = a.accumulate ? o[j] + v[j] : v[j];
    }
  }
  if (split > 1) cluster_sync_all();  // no CTA leaves while another still reads its shared memory
}

// ---------------------------------------------------------------------------
// CTA-pair kernel
// ---------------------------------------------------------------------------
constexpr int kPairStages = 6, kPairHalf = 128 * 64 * 2, kPairStage = 2 * kPairHalf;
constexpr int kTurnBytes = 32 * 128;  // a warp's 32 x 32 floats, turned on their way out
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + 256 /*barriers*/ + 256 /*unit sums*/ + 8 * kTurnBytes;

__device__ __forceinline__ float added(float a, float b) { return a + b; }
__device__ __forceinline__ float4 added(const float4& a, const float4& b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
// Stores (or adds) a warp's turned 32 x 32 floats to the rows at o, V at a time: each access of the warp covers whole lines of
// one row (float) or four (float4), where each lane storing its own row touched 32 lines (4096 x 8192, 256 chains: 76 us, now
// 39).  What is added to is read a batch ahead of its stores, which would otherwise order every read behind the store before
// it (adding to 4096 x 8192 floats, 256 chains: 192 us, now 91; to 4096 x 8191, 1024 chains: 409 us, now 151).
template <typename V>
__device__ __forceinline__ void put_rows(const unsigned char* turn, float* o, int64_t ld, int rows, int live, bool add) {
  constexpr int kPerRow = 128 / (int)sizeof(V), kRows = 32 / kPerRow, kBatch = sizeof(V) == 16 ? 4 : 8;
  const int lane = threadIdx.x & 31, k = lane % kPerRow * (int)sizeof(V);
  if (k / 4 >= live) return;
  o += k / 4;
  auto staged = [&](int r) {
    return *reinterpret_cast<const V*>(turn + r * 128 + ((k & ~15) ^ ((r & 7) << 4)) + (k & 15));
  };
  int r0 = lane / kPerRow;
  if (!add) {
#pragma unroll 8
    for (int r = r0; r < rows; r += kRows) *reinterpret_cast<V*>(o + (int64_t)r * ld) = staged(r);
    return;
  }
#pragma unroll 1
  for (; r0 < rows; r0 += kBatch * kRows) {
    V old[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      old[i] = *reinterpret_cast<const V*>(o + (int64_t)min(r0 + i * kRows, rows - 1) * ld);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = r0 + i * kRows;
      if (r < rows) *reinterpret_cast<V*>(o + (int64_t)r * ld) = added(staged(r), old[i]);
    }
  }
}

// Tile t -> (m, n) block: `group` row blocks at a time, row-fastest, so that the tiles in flight form a rectangle and
// share their operands' panels in L2.
__device__ __forceinline__ void pair_tile(const MomentArgs& a, int t, int& mb, int& nb) {
  const int m_blocks = (a.M + 255) / 256, n_blocks = (a.N + 255) / 256;
  const int per = a.group * n_blocks, g = t / per, w = t - g * per;
  const int rows = min(a.group, m_blocks - g * a.group);
  mb = g * a.group + w % rows;
  nb = w / rows;
}

__global__ void __launch_bounds__(kMomentThreads, 1)
    k_pair_moments_2sm(const __grid_constant__ MomentMaps maps, const __grid_constant__ MomentArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + kPairStages * kPairStage);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* side = reinterpret_cast<float*>(tiles + kPairStages * kPairStage + 256);
  if ((int)blockIdx.x >= a.tile_blocks) {  // whole clusters
    wait_for_previous_kernel();
    own_sums(a, reinterpret_cast<float*>(tiles));
    return;
  }

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = ((a.M + 255) / 256) * ((a.N + 255) / 256);
  const int first = (int)cluster_id_x(), step = a.tile_blocks / 2;
  const int total = a.total_blocks;  // > 0

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);  // every accumulating warp of both CTAs
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
  wait_for_previous_kernel();
  int last_chunk[2] = {-1, -1};

  if (warp == 0) {  // producer (both CTAs): this CTA's halves of the x and y units
    const bool one = elect_one();
    int64_t issued = 0;
    bool failed = false;
    for (int t = first; t < n_tiles && !failed; t += step) {
      int mb, nb;
      pair_tile(a, t, mb, nb);
      const int m0 = mb * 256 + (int)rank * 128, n0 = nb * 256 + (int)rank * 128;
      for (int b = 0; b < total && !failed;) {
        const Chunk c = chunk_at(a, b, total);
        for (int i = 0; i < c.length; ++i, ++issued) {
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
            const int chain = (c.block + i) * 64;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              tma_load_2d_pair(st + k * 8192, &maps.x[c.phase], bar, m0 + 64 * k, chain);
              tma_load_2d_pair(st + kPairHalf + k * 8192, &maps.y[c.phase], bar, n0 + 64 * k, chain);
            }
          }
          __syncwarp();
        }
        b += c.length;
      }
    }
    // every stage this CTA filled has been consumed (released by the leader's MMAs) before exit
    for (int64_t j = issued > kPairStages ? issued - kPairStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&empty[j % kPairStages], (uint32_t)(j / kPairStages) & 1u) && one) atomicExch(a.error, kErrEmptyWait);
  } else if (warp == 1) {
    if (leader) {  // MMA issue: the leader only
      const bool one = elect_one();
      const uint32_t idesc = (idesc_moments(256, a.f16 != 0) & 0x00FFFFFFu) | (16u << 24);  // M = 256
      int64_t used = 0;
      int chunk = 0;
      bool failed = false;
      for (int t = first; t < n_tiles && !failed; t += step) {
        for (int b = 0; b < total && !failed; ++chunk) {
          const Chunk c = chunk_at(a, b, total);
          const int buf = chunk & 1;
          if (!mbar_wait_all(&acc_empty[buf], ((uint32_t)(chunk >> 1) & 1u) ^ 1u)) {
            if (one) atomicExch(a.error, kErrAccWait);
            failed = true;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(buf * 256);
          for (int i = 0; i < c.length; ++i, ++used) {
            const int s = (int)(used % kPairStages);
            if (!mbar_wait_all(&full[s], (uint32_t)(used / kPairStages) & 1u)) {
              if (one) atomicExch(a.error, kErrFullWait);
              failed = true;
              break;
            }
            tc_fence_after();
            const unsigned char* st = tiles + s * kPairStage;
            const uint64_t ad = umma_desc_mn128(st), bd = umma_desc_mn128(st + kPairHalf);
            if (one) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)  // 16 chains per MMA: two groups of eight, 2048 bytes
                umma_f16_pair(d, ad + 128ull * kk, bd + 128ull * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
              umma_commit_pair(&empty[s]);  // the stage is free again in both CTAs
            }
            __syncwarp();
          }
          if (one) umma_commit_pair(&acc_full[buf]);  // both CTAs' accumulator halves complete
          __syncwarp();
          last_chunk[buf] = chunk;
          b += c.length;
        }
      }
    }
  } else if (warp >= 10) {
    side_sums(a, side);
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    unsigned char* turn = tiles + kPairStages * kPairStage + 512 + (warp - 2) * kTurnBytes;
    int chunk = 0;
    bool failed = false;
    for (int t = first; t < n_tiles && !failed; t += step) {
      int mb, nb;
      pair_tile(a, t, mb, nb);
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
      for (int b = 0; b < total; ++chunk) {
        const Chunk c = chunk_at(a, b, total);
        const int buf = chunk & 1;
        if (!mbar_wait_warp(&acc_full[buf], (uint32_t)(chunk >> 1) & 1u)) {
          if (lane == 0) atomicExch(a.error, kErrAccWait);
          failed = true;
          break;
        }
        tc_fence_after();
        const float scale = a.scale[c.phase];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[32];
          tmem_load32(tmem + (uint32_t)(buf * 256 + half * 128 + q * 32) + ((uint32_t)(quad * 32) << 16), v);
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[q * 32 + j] = fmaf(scale, v[j], acc[q * 32 + j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(&acc_empty[buf]);
        b += c.length;
      }
      if (failed) break;
      const int m0 = mb * 256 + (int)rank * 128 + quad * 32, n = nb * 256 + half * 128;
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // 32 columns of the warp's 32 rows at a time
        const int live = min(32, a.N - n - q * 32), rows = min(32, a.M - m0);
#pragma unroll
        for (int j = 0; j < 8; ++j)  // piece j of row r lies at j ^ (r & 7): rows and columns both cover every bank
          *reinterpret_cast<float4*>(turn + lane * 128 + 16 * (j ^ (lane & 7))) =
              make_float4(acc[q * 32 + 4 * j], acc[q * 32 + 4 * j + 1], acc[q * 32 + 4 * j + 2], acc[q * 32 + 4 * j + 3]);
        __syncwarp();
        float* o = a.out + (int64_t)m0 * a.out_ld + n + q * 32;
        if (a.vector_store && live == 32)
          put_rows<float4>(turn, o, a.out_ld, rows, live, a.accumulate != 0);
        else
          put_rows<float>(turn, o, a.out_ld, rows, live, a.accumulate != 0);
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1 && leader) {
    // every MMA the pair issued has completed (in both CTAs' TMEM) before TMEM is freed
    if (lane == 0) {
      for (int b = 0; b < 2; ++b)
        if (last_chunk[b] >= 0) (void)mbar_wait(&acc_full[b], (uint32_t)(last_chunk[b] >> 1) & 1u);
    }
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA frees TMEM or exits while the other may still signal it
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Tensor map of a chain-major 16-bit matrix [chains][units], read in boxes of 64 chains x 64 units, 128-byte swizzle.
int make_map_units(CUtensorMap* map, const void* base, int64_t chains, int64_t units, int64_t ld, bool f16) {
  EncodeTiledFn fn;
  int rc = encode_fn(&fn);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)units, (cuuint64_t)chains};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64u, 64u};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for a %lld x %lld 16-bit matrix", (int)r, (long long)chains,
              (long long)units);
    return TTHRML_ERR_CUDA;
  }
  return TTHRML_OK;
}

// Clusters of 1, 2, 4 and 8 CTAs of k_pair_moments<BN> that are resident at once on the current device.
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
    const int rc = cluster_fit((const void*)k_pair_moments<BN>, 1u << i, kMomentThreads, MomentShape<BN>::kSmem, &fit);
    if (rc) return rc;
    known[dev][i] = fit.clusters;
  }
  *out = known[dev];
  return TTHRML_OK;
}

// Estimated clocks of the tiles on clusters of S CTAs: per wave the blocks of a CTA's share of the chains (block_clocks), at
// least 360 clocks each to issue, the tile's store, and for S > 1 a barrier and the partial tiles.  The constants are those
// of the 8-bit tiles; over 28 sizes with every (BN, S) and the pair kernel measured, without unit sums and on rows that start
// on 16 bytes, the choice is 0.4 % behind the fastest on average, 7 % at most (777 x 2000 x 1523 chains: (128, 1) 12.1 us of
// 12.1 to 87; 512 x 1024 x 9216: (128, 4) 16.2 of 16.2 to 51; 1500 x 1500 x 5000: (256, 2) 26.0 of 26.0 to 150).  The unit
// sums are not counted.  Where the tiles leave a few SMs over, these take all strips and end long after the tiles: 2304 x
// 2048 x 9216 chains 62 us, with sums 760; 1500 x 1500 x 5000 157; 512 x 1024 x 9216 44; 4096 x 8192 x 9216 (no SM is left
// over) 444 and 468.
template <int BN>
int consider(const MomentArgs& a, int64_t& best, int& bn, int& split) {
  const int* resident;
  const int rc = resident_tiles<BN>(&resident);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  for (int i = 0; i < 4 && (i == 0 || (1 << i) <= a.total_blocks); ++i) {
    const int s = 1 << i;
    const int64_t waves = (tiles + resident[i] - 1) / resident[i];
    const int64_t block =
        block_clocks(MomentShape<BN>::kStage, (tiles < resident[i] ? tiles : resident[i]) * s, std::max(2 * BN, 360));
    const int64_t c = 8300 + waves * ((int64_t)((a.total_blocks + s - 1) / s) * block + 20 * BN + (s > 1 ? 850 + 128 * BN / 10 : 0));
    if (c < best) best = c, bn = BN, split = s;
  }
  return TTHRML_OK;
}

template <int BN>
int launch_tiles(const MomentMaps& maps, MomentArgs& a, int split, int sms, bool early, cudaStream_t st) {
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN) * split;
  a.tile_blocks = (int32_t)tiles;
  // CTAs of their own for the unit sums where SMs are left over, else the tiles' CTAs take them along
  // (a strip is a cluster's; clusters of 8 and of 4 leave some SMs of a GPU unused, so some of these may run late)
  const int64_t strips = sum_strips(a), left = tiles < sms ? (sms - tiles) / split : 0;
  const int64_t grid = tiles + (strips > 0 && left > 0 ? (strips < left ? strips : left) * split : 0);
  void* params[2] = {(void*)&maps, (void*)&a};
  return launch_clusters((const void*)k_pair_moments<BN>, (unsigned)grid, (unsigned)split, kMomentThreads,
                         MomentShape<BN>::kSmem, params, st, "k_pair_moments launch", early);
}

int launch_moments(const MomentMaps& maps, MomentArgs& a, bool early, cudaStream_t st) {
  ClusterFit fit;
  int rc = cluster_fit((const void*)k_pair_moments_2sm, 2, kMomentThreads, kPairSmem, &fit);
  if (rc) return rc;
  int64_t best = INT64_MAX;
  int bn = 128, split = 1;
  if ((rc = consider<64>(a, best, bn, split)) || (rc = consider<128>(a, best, bn, split)) ||
      (rc = consider<256>(a, best, bn, split)))
    return rc;
  const int64_t mblk = (a.M + 255) / 256, nblk = (a.N + 255) / 256, pairs = mblk * nblk;
  // the pair kernel overlaps a tile's store with the next tile's loop
  const int64_t waves = (pairs + fit.clusters - 1) / fit.clusters;
  const int64_t block = block_clocks(kPairStage, 2 * (pairs < fit.clusters ? pairs : fit.clusters), 684);
  const int64_t clocks = 13700 + waves * ((int64_t)a.total_blocks * block + 3000);
  if (a.total_blocks > 0 && clocks < best) {
    int64_t g = 1;  // about square rectangles of the tiles in flight
    while ((g + 1) * (g + 1) <= fit.clusters) ++g;
    a.group = (int32_t)(g < mblk ? g : mblk);
    const int64_t clusters = pairs < fit.clusters ? pairs : fit.clusters;
    a.tile_blocks = (int32_t)(2 * clusters);
    // clusters of their own for the unit sums where SMs are left over, else warps of the tiles' CTAs take them along
    const int64_t want = sum_strips(a), left = fit.clusters - clusters;
    const int64_t others = want < left ? want : left;
    void* params[2] = {(void*)&maps, (void*)&a};
    return launch_clusters((const void*)k_pair_moments_2sm, (unsigned)(2 * (clusters + others)), 2, kMomentThreads, kPairSmem,
                           params, st, "k_pair_moments_2sm launch", early);
  }
  if (bn == 64) return launch_tiles<64>(maps, a, split, fit.sms, early, st);
  if (bn == 128) return launch_tiles<128>(maps, a, split, fit.sms, early, st);
  return launch_tiles<256>(maps, a, split, fit.sms, early, st);
}

// Rows of 16-bit elements from any strides to rows that start on 16 bytes, several matrices in one launch
// (blockIdx.y): eight elements per thread, columns behind the end as zeros.  Adjacent elements are read as aligned words.
struct PackArgs {
  tthrml_pack_matrix m[TTHRML_MAX_PACKED];
};
__global__ void __launch_bounds__(256) k_pack_rows(const __grid_constant__ PackArgs a) {
  let_next_kernel_start();
  const tthrml_pack_matrix& m = a.m[blockIdx.y];
  const uint32_t per_row = (uint32_t)(m.pitch / 8);
  const uint32_t rows_at_once = per_row >= 256u ? 1u : 256u / per_row;  // rows that a block takes side by side
  const uint32_t t_row = threadIdx.x / per_row, t_vec = threadIdx.x - t_row * per_row;
  if (per_row < 256u && t_row >= rows_at_once) return;
  const int64_t step = (int64_t)gridDim.x * rows_at_once;
  for (int64_t row0 = (int64_t)blockIdx.x * rows_at_once + (per_row < 256u ? t_row : 0u); row0 < m.rows; row0 += 4 * step) {
    for (uint32_t v = per_row < 256u ? t_vec : threadIdx.x; v < per_row; v += 256u) {
      const int64_t c = (int64_t)v * 8;
      uint4 out[4];  // four rows on their way at a time
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t row = row0 + j * step;
        if (row >= m.rows) break;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(m.src) + row * m.row_stride;
        if (m.col_stride == 1 && c + 8 <= m.cols) {
          // the words that hold the eight elements; a fifth one where the first element is the upper half of a word
          const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)(src + c) & ~(uintptr_t)3);
          const bool odd = ((uintptr_t)(src + c) & 2) != 0;
          const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = odd ? w[4] : 0u;
          out[j] = odd ? make_uint4(__funnelshift_r(w0, w1, 16), __funnelshift_r(w1, w2, 16), __funnelshift_r(w2, w3, 16),
                                    __funnelshift_r(w3, w4, 16))
                       : make_uint4(w0, w1, w2, w3);
        } else {
          uint32_t e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = c + i < m.cols ? src[(c + i) * m.col_stride] : 0u;
          out[j] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t row = row0 + j * step;
        if (row < m.rows) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(m.dst) + row * m.pitch + c) = out[j];
      }
    }
  }
}

}  // namespace
}  // namespace tthrml

namespace {

// early: the operands were laid out by the kernel just before on the stream
int pair_moments(const tthrml_moment_phase* phases_host, int32_t n_phases, int32_t dtype, int64_t x_units, int64_t y_units,
                 float* out, int64_t out_ld, float* x_sum, float* y_sum, int32_t accumulate, int32_t* error, bool early,
                 void* stream) {
  using namespace tthrml;
  if (x_units == 0 && y_units == 0) return TTHRML_OK;
  if (!phases_host || !out || !error) {
    set_error("tthrml_pair_moments: NULL argument");
    return TTHRML_ERR_ARG;
  }
  if (n_phases < 1 || n_phases > TTHRML_MAX_PHASES) {
    set_error("tthrml_pair_moments: 1 to %d phases are supported (got %d)", TTHRML_MAX_PHASES, (int)n_phases);
    return TTHRML_ERR_ARG;
  }
  if (dtype != TTHRML_DT_BF16 && dtype != TTHRML_DT_F16) {
    set_error("tthrml_pair_moments: elements must be bfloat16 or float16 (got code %d)", (int)dtype);
    return TTHRML_ERR_ARG;
  }
  if (x_units < 1 || y_units < 1 || x_units > 0x3fffffffLL || y_units > 0x3fffffffLL || out_ld < y_units ||
      ((x_units + 127) / 128) * ((y_units + 63) / 64) > 0x0fffffffLL) {
    set_error("tthrml_pair_moments: sizes out of range (%lld x %lld units, output pitch %lld)", (long long)x_units,
              (long long)y_units, (long long)out_ld);
    return TTHRML_ERR_ARG;
  }
  MomentMaps maps;
  MomentArgs a;
  a.n_phases = n_phases;
  a.total_blocks = 0;
  for (int p = 0; p < TTHRML_MAX_PHASES; ++p) {
    const tthrml_moment_phase& h = phases_host[p < n_phases ? p : 0];
    if (p >= n_phases) {  // never read
      maps.x[p] = maps.x[0];
      maps.y[p] = maps.y[0];
      a.x[p] = a.y[p] = nullptr;
      a.x_ld[p] = a.y_ld[p] = a.chains[p] = 0;
      a.blocks[p] = 0;
      a.scale[p] = a.x_scale[p] = a.y_scale[p] = 0.0f;
      continue;
    }
    if (h.chains < 0 || h.chains > 0x3fffffffLL || (h.chains > 0 && (!h.x || !h.y)) || (uintptr_t)h.x % 16 ||
        (uintptr_t)h.y % 16 || h.x_ld % 8 || h.y_ld % 8 || h.x_ld < x_units || h.y_ld < y_units) {
      set_error("tthrml_pair_moments: phase %d: operands must be 16-byte aligned with pitches that are multiples of 8 "
                "elements and not below the units (got %lld chains, pitches %lld, %lld)", p, (long long)h.chains,
                (long long)h.x_ld, (long long)h.y_ld);
      return TTHRML_ERR_ARG;
    }
    a.x[p] = h.x;
    a.y[p] = h.y;
    a.x_ld[p] = h.x_ld;
    a.y_ld[p] = h.y_ld;
    a.chains[p] = h.chains;
    a.blocks[p] = (int32_t)((h.chains + 63) / 64);
    a.scale[p] = h.scale;
    a.x_scale[p] = h.x_scale;
    a.y_scale[p] = h.y_scale;
    if ((int64_t)a.total_blocks + a.blocks[p] > 0x3fffffffLL) {
      set_error("tthrml_pair_moments: too many chains");
      return TTHRML_ERR_ARG;
    }
    a.total_blocks += a.blocks[p];
  }
  for (int p = 0; p < n_phases; ++p) {
    if (!a.chains[p]) continue;
    int rc = make_map_units(&maps.x[p], a.x[p], a.chains[p], x_units, a.x_ld[p], dtype == TTHRML_DT_F16);
    if (rc == TTHRML_OK) rc = make_map_units(&maps.y[p], a.y[p], a.chains[p], y_units, a.y_ld[p], dtype == TTHRML_DT_F16);
    if (rc) return rc;
  }
  a.M = (int32_t)x_units;
  a.N = (int32_t)y_units;
  a.out = out;
  a.out_ld = out_ld;
  a.x_sum = x_sum;
  a.y_sum = y_sum;
  a.accumulate = accumulate != 0;
  a.vector_store = (uintptr_t)out % 16 == 0 && out_ld % 4 == 0;
  a.f16 = dtype == TTHRML_DT_F16;
  a.error = error;
  return launch_moments(maps, a, early, (cudaStream_t)stream);
}

}  // namespace

extern "C" int tthrml_pair_moments(const tthrml_moment_phase* phases_host, int32_t n_phases, int32_t dtype,
                                   int64_t x_units, int64_t y_units, float* out, int64_t out_ld, float* x_sum,
                                   float* y_sum, int32_t accumulate, int32_t* error, void* stream) {
  return pair_moments(phases_host, n_phases, dtype, x_units, y_units, out, out_ld, x_sum, y_sum, accumulate, error, false,
                      stream);
}

extern "C" int tthrml_pair_moments_packed(const tthrml_pack_matrix* matrices_host, int32_t n_matrices,
                                          const tthrml_moment_phase* phases_host, int32_t n_phases, int32_t dtype,
                                          int64_t x_units, int64_t y_units, float* out, int64_t out_ld, float* x_sum,
                                          float* y_sum, int32_t accumulate, int32_t* error, void* stream) {
  const int rc = tthrml_pack_rows(matrices_host, n_matrices, stream);
  if (rc) return rc;
  bool packed = false;  // whether a kernel was launched
  for (int i = 0; i < n_matrices; ++i) packed = packed || matrices_host[i].rows > 0;
  return pair_moments(phases_host, n_phases, dtype, x_units, y_units, out, out_ld, x_sum, y_sum, accumulate, error, packed,
                      stream);
}

extern "C" int tthrml_pack_rows(const tthrml_pack_matrix* matrices_host, int32_t n, void* stream) {
  using namespace tthrml;
  if (n == 0) return TTHRML_OK;
  if (!matrices_host || n < 0 || n > TTHRML_MAX_PACKED) {
    set_error("tthrml_pack_rows: 0 to %d matrices are supported (got %d)", TTHRML_MAX_PACKED, (int)n);
    return TTHRML_ERR_ARG;
  }
  PackArgs a = {};
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    const tthrml_pack_matrix& m = matrices_host[i];
    if (m.rows < 0 || m.cols < 1 || m.pitch < m.cols || m.pitch % 8 || m.pitch > 0x7fffffffLL || m.row_stride < 0 ||
        m.col_stride < 0 || (m.rows > 0 && (!m.src || !m.dst || (uintptr_t)m.src % 2 || (uintptr_t)m.dst % 16))) {
      set_error("tthrml_pack_rows: matrix %d: %lld x %lld, pitch %lld (a multiple of 8), targets 16-byte aligned", i,
                (long long)m.rows, (long long)m.cols, (long long)m.pitch);
      return TTHRML_ERR_ARG;
    }
    a.m[i] = m;
    const int64_t at_once = 4 * (m.pitch / 8 >= 256 ? 1 : 256 / (m.pitch / 8)), blocks = (m.rows + at_once - 1) / at_once;
    most = blocks > most ? blocks : most;
  }
  if (most == 0) return TTHRML_OK;
  const int64_t limit = 148 * 8;
  k_pack_rows<<<dim3((unsigned)(most < limit ? most : limit), (unsigned)n), 256, 0, (cudaStream_t)stream>>>(a);
  return launch_status("k_pack_rows launch");
}
