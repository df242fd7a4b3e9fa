// Pair moments of two blocks over the chain batch, on the tensor cores (tcgen05.mma kind::f16):
//     out[i][j] (+)= sum_p s_p sum_c x_p[c][i] y_p[c][j],   with the unit sums sum_p s_p sum_c x_p[c][i] (and y).
// With a data phase (s = -1 / chains) and a model phase (s = 1 / chains) this is the gradient of a dense program's
// couplings and biases (the likelihood gradient of a Boltzmann machine; Ackley, Hinton and Sejnowski 1985).
//
// Both operands lie chain-major (the layout of the sampler's states), so the sum runs over the slow axis of each:
// the tiles are MN-major in shared memory (64 units x 64 chains per TMA box, 128-byte swizzle) and nothing is
// transposed.  A cluster of S CTAs computes one 128 x BN tile, each CTA a contiguous share of the 64-chain blocks:
//   warp 0    TMA loads into a ring of stages (chains and units behind the ends read as zeros);
//   warp 1    MMAs, kChunk blocks (512 chains) into one of two TMEM accumulators;
//   warps 2-9 add each finished accumulator, times its phase's scale, to float32 registers (BN / 2 per thread).
// The tensor core's accumulation drops bits over long sums, so a sum longer than 512 chains is carried in registers with
// rounded float32 additions.  The S partial tiles are added over distributed shared memory in the order of the ranks, so
// the result is the same every time.  Blocks behind the tiles sum the units.
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace tthrml {
namespace {

constexpr int kMomentThreads = 320;
constexpr int kChunkBlocks = 8;     // 64-chain blocks per TMEM accumulation
constexpr int kSumUnits = 32;       // units per block of unit sums

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
  int32_t tile_blocks; // CTAs that compute tiles; the others sum units
  int* error;
};

template <int BN>
struct MomentShape {
  static constexpr int kABytes = 128 * 64 * 2, kBBytes = BN * 64 * 2;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int kPitch = BN + 4;
  static constexpr int kSmem = 1024 + kStages * kStage + 256;
  static_assert(128 * kPitch * 4 <= kStages * kStage, "the staged tile reuses the operand stages");
};

// Shared-memory descriptor of an MN-major tile in the 128-byte swizzle: boxes of 64 units x 64 chains (8 KiB), so
// groups of 64 units are 8192 bytes apart (leading offset) and groups of 8 chains 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t umma_desc_mn128(const void* tile) {
  const uint64_t addr = (uint64_t)(smem_u32(tile) >> 4) & 0x3FFFull;
  return addr | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// D float32, A and B bfloat16 (or float16), both MN-major.
__device__ __forceinline__ uint32_t idesc_moments(int n, bool f16) {
  const uint32_t t = f16 ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
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

// Unit sums of units u0 .. u0 + 31 of x (or y) by one CTA: a thread takes two adjacent units of every 20th chain, then
// the partial sums are added in the order of the chains' lanes.
__device__ void unit_sums(const MomentArgs& a, bool of_y, int u0, float* part) {
  constexpr int kLanes = kMomentThreads / (kSumUnits / 2);  // 20 chain lanes
  const int u = (threadIdx.x % (kSumUnits / 2)) * 2, lane = threadIdx.x / (kSumUnits / 2);
  const int units = of_y ? a.N : a.M;
  float t0 = 0.0f, t1 = 0.0f;
  for (int p = 0; p < a.n_phases; ++p) {
    const void* base = of_y ? a.y[p] : a.x[p];
    const int64_t ld = of_y ? a.y_ld[p] : a.x_ld[p];
    const float scale = of_y ? a.y_scale[p] : a.x_scale[p];
    if (scale == 0.0f) continue;
    float s0 = 0.0f, s1 = 0.0f;
    if (u0 + u + 2 <= units) {  // rows start on 16 bytes, units on even places: a 4-byte load
#pragma unroll 8
      for (int64_t c = lane; c < a.chains[p]; c += kLanes) {
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(base) + (c * ld + u0 + u) / 2);
        if (a.f16) {
          const __half2 h = *reinterpret_cast<const __half2*>(&w);
          s0 += __low2float(h);
          s1 += __high2float(h);
        } else {
          s0 += __uint_as_float(w << 16);
          s1 += __uint_as_float(w & 0xFFFF0000u);
        }
      }
    } else if (u0 + u < units) {
      for (int64_t c = lane; c < a.chains[p]; c += kLanes) s0 += elem(base, c * ld + u0 + u, a.f16 != 0);
    }
    t0 = fmaf(scale, s0, t0);
    t1 = fmaf(scale, s1, t1);
  }
  part[lane * kSumUnits + u] = t0;
  part[lane * kSumUnits + u + 1] = t1;
  __syncthreads();
  if (threadIdx.x < kSumUnits && u0 + (int)threadIdx.x < units) {
    float s = 0.0f;
    for (int i = 0; i < kLanes; ++i) s += part[i * kSumUnits + threadIdx.x];
    float* dst = (of_y ? a.y_sum : a.x_sum) + u0 + threadIdx.x;
    *dst = a.accumulate ? *dst + s : s;
  }
}

template <int BN>
__global__ void __launch_bounds__(kMomentThreads, 1)
    k_pair_moments(const __grid_constant__ MomentMaps maps, const __grid_constant__ MomentArgs a) {
  using S = MomentShape<BN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  if ((int)blockIdx.x >= a.tile_blocks) {  // whole clusters: the tile blocks are a multiple of the cluster size
    const int strip = (int)blockIdx.x - a.tile_blocks, xs = a.x_sum ? (a.M + kSumUnits - 1) / kSumUnits : 0;
    const int ys = a.y_sum ? (a.N + kSumUnits - 1) / kSumUnits : 0;
    if (strip < xs)
      unit_sums(a, false, strip * kSumUnits, reinterpret_cast<float*>(tiles));
    else if (strip - xs < ys)
      unit_sums(a, true, (strip - xs) * kSumUnits, reinterpret_cast<float*>(tiles));
    return;
  }
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S::kStages * S::kStage);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);

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

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      bool failed = false;
      for (int b = first; b < last && !failed;) {
        const Chunk c = chunk_at(a, b, last);
        for (int i = 0; i < c.length; ++i, ++issued) {
          const int s = issued % S::kStages;
          if (!mbar_wait(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
            atomicExch(a.error, kErrEmptyWait);
            failed = true;
            break;
          }
          mbar_expect_tx(&full[s], S::kStage);
          unsigned char* t = tiles + s * S::kStage;
          const int chain = (c.block + i) * 64;
#pragma unroll
          for (int k = 0; k < 2; ++k) tma_load_2d(t + k * 8192, &maps.x[c.phase], &full[s], m0 + 64 * k, chain);
#pragma unroll
          for (int k = 0; k < BN / 64; ++k)
            tma_load_2d(t + S::kABytes + k * 8192, &maps.y[c.phase], &full[s], n0 + 64 * k, chain);
        }
        b += c.length;
      }
      // the copies issued must land before the stages are used again or the CTA exits
      for (int j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
        if (!mbar_wait(&full[j % S::kStages], (uint32_t)(j / S::kStages) & 1u)) atomicExch(a.error, kErrFullWait);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_moments(BN, a.f16 != 0);
      int used = 0, chunk = 0;
      bool failed = false;
      for (int b = first; b < last && !failed; ++chunk) {
        const Chunk c = chunk_at(a, b, last);
        const int buf = chunk & 1;
        if (!mbar_wait(&acc_empty[buf], ((uint32_t)(chunk >> 1) & 1u) ^ 1u)) {
          atomicExch(a.error, kErrAccWait);
          failed = true;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * BN);
        for (int i = 0; i < c.length; ++i, ++used) {
          const int s = used % S::kStages;
          if (!mbar_wait(&full[s], (uint32_t)(used / S::kStages) & 1u)) {
            atomicExch(a.error, kErrFullWait);
            failed = true;
            break;
          }
          tc_fence_after();
          const unsigned char* t = tiles + s * S::kStage;
          const uint64_t ad = umma_desc_mn128(t), bd = umma_desc_mn128(t + S::kABytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 chains per MMA: two groups of eight, 2048 bytes
            umma_f16(d, ad + 128ull * kk, bd + 128ull * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        umma_commit(&acc_full[buf]);
        b += c.length;
      }
    }
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
      if (!mbar_wait(&acc_full[buf], (uint32_t)(chunk >> 1) & 1u)) {
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

template <int BN>
int launch_moments(const MomentMaps& maps, MomentArgs a, int split, cudaStream_t st) {
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  a.tile_blocks = (int32_t)(tiles * split);
  const int64_t strips = (a.x_sum ? (a.M + kSumUnits - 1) / kSumUnits : 0) + (a.y_sum ? (a.N + kSumUnits - 1) / kSumUnits : 0);
  const int64_t grid = tiles * split + (strips + split - 1) / split * split;
  void* params[2] = {(void*)&maps, (void*)&a};
  return launch_clusters((const void*)k_pair_moments<BN>, (unsigned)grid, (unsigned)split, kMomentThreads,
                         MomentShape<BN>::kSmem, params, st, "k_pair_moments launch");
}

}  // namespace
}  // namespace tthrml

extern "C" int tthrml_pair_moments(const tthrml_moment_phase* phases_host, int32_t n_phases, int32_t dtype,
                                   int64_t x_units, int64_t y_units, float* out, int64_t out_ld, float* x_sum,
                                   float* y_sum, int32_t accumulate, int32_t* error, void* stream) {
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
  cudaStream_t st = (cudaStream_t)stream;
  if (y_units > 128) return launch_moments<256>(maps, a, 1, st);
  return launch_moments<128>(maps, a, 1, st);
}
