// Softmax cross entropy over a large set of categories on the tensor cores, in pieces, without keeping the logits:
//     l[t][v] = sum_k x[t][k] w[v][k] + b[v],   z[t] = log sum_v exp l[t][v],   loss[t] = z[t] - l[t][y[t]],
// and, with r[t] the weight of row t in what is differentiated,
//     g[t][v] = r[t] (exp(l[t][v] - z[t]) - [v == y[t]]),   dx = g w,   dw = g^T x,   db = sum_t g.
//
// The forward pass is one product whose epilogue folds each tile of logits into a running maximum and sum per row (a row
// per thread; log2 domain), so only a pair of floats per row and unit of work leaves the SM; k_xent_loss joins them.  The
// backward pass takes the categories in pieces of kPieceBytes of g, of 256 categories at least: the logits of a piece are computed again and
// turned into g (16 bits), which two further products reduce to this piece's rows of dw and to sums of dx in float32.
//
// One kernel serves the four products: persistent clusters of two CTAs walk 256 x BN tiles (tcgen05 cta_group::2, two
// TMEM accumulators, four to eight stages of 64 columns of K), operands K-major or MN-major as they lie in memory, so nothing is
// transposed.  Warps 2 on run the epilogue of a tile beside the main loop of the next one: eight, or sixteen where the logits are
// short sums or db is summed up beside.  Logits of up to 128 rows are tiles of one CTA each: a pair's MMA would take as long for
// half the weights, which are what bounds them (64 rows, 4096 x 32768 weights: 58 us in pairs).  Warp 0 loads (TMA), warp 1 of the
// even CTA multiplies.
//
// g is rounded to the operands' 16 bits (up to kFewRows rows or kFewCategories categories: held in two such pieces, their sum
// good to 2^-16; the second piece is more rows or columns of the same tiles): by at most 2^-8 (bfloat16) or 2^-11 (float16) of
// each element, as dx and dw themselves are.  float16 holds g times 2^14 over the largest weight of a row, so that what is at least 2^-28 of
// that weight stays a normal number and rows of far smaller weights lose bits.  Maxima and sums are float32, as dx and dw accumulate; losses and
// the sums of db are joined in 64 bits and leave as float32.
//
// What bounds it: the tensor pipe (97 % active, in g 87 %; 4096 rows, 4096 columns, 16384 categories: logits 332 us, g 373 (its epilogue is
// longer than the two accumulations that run ahead of it), dx 383, dw 344, 1.43 to 1.65 PFLOP/s at the clocks of a short run) and, over
// longer runs, the power cap (8192 x 4096 x 32768, the whole step: 6.7 to 7.0 ms, 1.25 to 1.32 PFLOP/s); the weights' bytes for few rows.
#include "int8_common.cuh"
#include "tc_common.cuh"

namespace tthrml {
namespace {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr int64_t kPieceBytes = 256ll << 20;  // of g at a time, or 256 categories (128 columns of two pieces) where those are more
// The products take g in 16 bits.  Where few of its values meet in a sum, their roundings' errors do not average out, and g is held
// in two pieces, the rounding's remainder the second: below the first rows, or beside the first columns.  (64 columns are one block of
// the sum for dx, 128 half a tile's rows for dw: the products take as long.)
constexpr int64_t kFewRows = 128, kFewCategories = 64;
// 64-wide blocks of K that a logit's sum stays in tensor memory for.  The tensor core cuts its sums off instead of rounding them;
// float32 registers add them up every few blocks, in both passes the same, so that probabilities and normalisers agree (a backward pass of
// one accumulation, which is quicker by 33 us of the 373 above, makes the difference of a row of probability 1 - 1e-4 wrong by a
// multiple of itself).  Errors of
// losses and db over 150 random sizes of 8 to 8192 columns, relative: four below 3e-7, eight below 5e-7, 32 some of 3e-6 (eight after
// four 1e-6).  Two, four and eight take 1.67, 1.53 and 1.36 ms for the losses of 8192 x 4096 x 32768, four and eight 62 and 59 us for
// those of 64 rows; fewer are taken where few rows meet few categories: nothing averages the errors out, and the time is not the
// tiles' (db of 13 x 409 x 2: 1.1e-7, 1.4e-7 and 1.8e-7 in the middle of 200 inputs with one, two and four, and 1.0e-7 in plain
// float32; a step of 100 x 8192 x 10 in 149, 118 and 103 us).  More categories average them out: 64 x 4096, losses of 128, 4096 and 32768
// categories off by up to 1.1e-7, 8e-8 and 7e-8 with four, 2.0e-7, 1.4e-7 and 1.2e-7 with eight, in 26.3, 27.1 and 56.5 us with four,
// 24.5, 25.2 and 56.8 with eight; 16384 categories in 47.0 and 43.3.
constexpr int chunk_of(int64_t rows, int64_t categories) {
  return rows > 128 || categories > 4096 ? 8 : (categories > 64 ? 4 : 2);
}
constexpr bool one_chunk(int64_t rows, int64_t categories, int64_t cols) { return (cols + 63) / 64 <= chunk_of(rows, categories); }
enum : int { kPartials = 0, kGradient = 1, kGradientSums = 2, kProduct = 3 };

struct RowTargets {
  const void* y;  // [rows] int64 or int32
  int32_t wide;
  int64_t ignored;
};
__device__ __forceinline__ int64_t target_of(const RowTargets& t, int64_t row) {
  return t.wide ? __ldg(reinterpret_cast<const long long*>(t.y) + row) : (int64_t)__ldg(reinterpret_cast<const int*>(t.y) + row);
}

struct XentArgs {
  int32_t M, N;       // the product's rows and columns
  int32_t num_k;      // 64-wide blocks of its sum
  int32_t f16;
  int32_t box_m;      // rows per load of A (16, 32, 64 or 128); those behind are whatever the stage held, and not used
  int32_t chunk;      // blocks of K per accumulation
  int32_t units, segments, seg, splits, group;  // units of work: `seg` tiles along N of one row of tiles and one share of K
  // epilogues of logits: N categories from `first` on
  const float* bias;  // of the first category, or NULL
  int64_t first, categories;  // of this piece, and of all
  RowTargets targets;
  // kPartials
  float2* part;       // [M][slots] (maximum, sum) in the log2 domain
  int32_t slots;
  float* target_logit;  // [M]
  uint32_t* counter;    // zeroed for k_xent_loss
  // kGradient
  const float2* sums;     // [M] (maximum, sum) over all categories
  const float* row_grad;  // [M] weights, or NULL: ones
  const float* top_grad;  // what they are divided by
  float unit;             // g is held times this
  float* bias_part;       // [ceil(M / 32)][bias_ld] sums over 32 rows, or NULL
  int64_t bias_ld;
  // kGradient: out = g.  kProduct: scaled, out = sums * factor[0] * factor[1] / unit; else planes of plain float32 sums, one per
  // split, added to where `accumulate`.  tma_store: `out` takes bulk stores (planes always do).
  void* out;
  int64_t out_ld;
  int32_t out_dtype, align, accumulate, scaled, tma_store;
  int32_t second;  // kGradient: the row of `out` where the remainders of the rounding begin, or 0.  kProduct: the block of K from
                   // which on B's rows begin again
  int32_t beside;  // kGradient: the column where they begin, all columns before and behind it written, or 0.  Neither: dropped
  const float* factor[2];
  const float* carry;  // kProduct, scaled: sums of earlier pieces to add, [M][carry_ld] with room for whole 32 columns
  int64_t carry_ld;
  int* error;
};

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float factor_of(const float* const (&f)[2]) {
  return (f[0] ? __ldg(f[0]) : 1.0f) * (f[1] ? __ldg(f[1]) : 1.0f);
}
// (m, s) stands for s 2^m; an empty sum has m = -inf and s = 0.  A NaN in s stays.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
  s = s * exp2_fast(m - base) + s2 * exp2_fast(m2 - base);
  m = top;
}

// Parts of a tile's columns that the epilogue's warps share: four warps, a row per lane, take one.
// Sixteen warps where the epilogue is what a tile waits for: beside short sums (one accumulation; losses of 8192 x 128 x 32768 in 105 us,
// 162 with eight) and with db's sums of columns (a step of 777 x 1008 x 5008: 77 us, 80 with eight).  Else eight do (losses of 8192 x
// 4096 x 32768 in 1.35 ms, 1.38 with sixteen).
constexpr int parts_of(bool brief, int bn, int epi = kPartials) { return (brief || epi == kGradientSums) && bn >= 128 ? 4 : 2; }
template <int EPI, int BN, int CTAS, bool BRIEF>
struct XentShape {
  static constexpr int kParts = parts_of(BRIEF, BN, EPI), kWarps = 4 * kParts, kThreads = 64 + 32 * kWarps;
  static constexpr int kA = 128 * 64 * 2, kB = BN / CTAS * 64 * 2, kStage = kA + kB;
  static constexpr int kOut = EPI == kProduct ? kWarps * kOutBytes : 0;  // rows on their way out
  static constexpr int kBarriers = 256;
  static constexpr int kMine = BN / kParts;  // columns of a warp
  static constexpr int kRest = 1024 + kOut + kBarriers + (EPI == kProduct ? 0 : kWarps * kMine * 4 /*their biases*/);
  static constexpr int kFit = (232448 - kRest) / kStage, kStages = kFit < 8 ? kFit : 8;
  static constexpr int kSmem = kRest + kStages * kStage;
};

// v less its values rounded to 16 bits (w, packed).
__device__ __forceinline__ void less_row(float (&v)[32], int32_t dtype, const uint4 (&w)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t p[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo, hi;
      if (dtype == TTHRML_DT_BF16) {
        lo = __uint_as_float(p[j] << 16), hi = __uint_as_float(p[j] & 0xFFFF0000u);
      } else {
        const __half2 h = *reinterpret_cast<const __half2*>(&p[j]);
        lo = __low2float(h), hi = __high2float(h);
      }
      v[8 * q + 2 * j] -= lo;
      v[8 * q + 2 * j + 1] -= hi;
    }
  }
}

// 32 bytes, a whole sector: a row per lane needs no turning in shared memory (8192 x 128 x 32768, a step: 544 us turned, 522 so).
__device__ __forceinline__ void store_sector(unsigned char* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
               "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (CTAS == 2)
    umma_commit_pair(bar);
  else
    umma_commit(bar);
}

// Unit u -> its split, row of tiles and segment: splits slowest, `group` rows of tiles at a time.
template <int ROWS>
__device__ __forceinline__ void unit_at(const XentArgs& a, int u, int& split, int& mb, int& sg) {
  const int m_blocks = (a.M + ROWS - 1) / ROWS, all = m_blocks * a.segments;
  split = u / all;
  const int t = u - split * all, per = a.group * a.segments, g = t / per, w = t - g * per;
  const int rows = min(a.group, m_blocks - g * a.group);
  mb = g * a.group + w % rows;
  sg = w / rows;
}

// Sums over the warp's 32 lanes of 32 values each: lane j returns that of value j.  (Turned in shared memory it takes 75
// instructions instead of 124, but the MMAs keep shared memory busy: db's pass of 4096 x 512 x 8192 in 47 us, so in 43.)
__device__ __forceinline__ float column_sums(const float (&v)[32]) {
  const uint32_t lane = threadIdx.x & 31;
  float s[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const bool up = lane & 16;
    const float mine = up ? v[j + 16] : v[j], other = up ? v[j] : v[j + 16];
    s[j] = mine + __shfl_xor_sync(0xffffffffu, other, 16);
  }
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
    for (int j = 0; j < w; ++j) {
      const bool up = lane & w;
      const float mine = up ? s[j + w] : s[j], other = up ? s[j] : s[j + w];
      s[j] = mine + __shfl_xor_sync(0xffffffffu, other, w);
    }
  return s[0];
}

template <int EPI, bool A_MN, bool B_MN, int BN, int CTAS, bool BRIEF>
__global__ void __launch_bounds__(XentShape<EPI, BN, CTAS, BRIEF>::kThreads, 1)
    k_xent(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
           const __grid_constant__ CUtensorMap map_out, const __grid_constant__ XentArgs a) {
  using S = XentShape<EPI, BN, CTAS, BRIEF>;
  constexpr int kRows = 128 * CTAS;  // of a tile
  static_assert(!B_MN || (BN == 256 && CTAS == 2), "MN-major halves of B are whole boxes of 64");
  constexpr bool kChunked = !BRIEF && EPI != kProduct;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* turns = tiles + S::kStages * S::kStage;  // a buffer per epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(turns + S::kOut);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* biases = reinterpret_cast<float*>(turns + S::kOut + S::kBarriers);  // [kWarps][kMine]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_blocks = (a.N + BN - 1) / BN;
  const int first = (int)cluster_id_x(), step = (int)n_clusters_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CTAS * S::kWarps);  // every epilogue warp of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  let_next_kernel_start();  // its setup beside this kernel; it waits for this one's end as this one does here
  wait_for_previous_kernel();
  if (EPI == kPartials && blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0u;
  int last_it[2] = {-1, -1};

  if (warp == 0) {  // producer (both CTAs): this CTA's halves of the A and B slices
    const bool one = elect_one();
    int64_t issued = 0;
    bool failed = false;
    for (int u = first; u < a.units && !failed; u += step) {
      int split, mb, sg;
      unit_at<kRows>(a, u, split, mb, sg);
      const int k_first = (int)((int64_t)a.num_k * split / a.splits), k_last = (int)((int64_t)a.num_k * (split + 1) / a.splits);
      const int m0 = mb * kRows + (int)rank * 128;
      for (int nb = sg * a.seg; nb < min((sg + 1) * a.seg, n_blocks) && !failed; ++nb) {
        const int n0 = nb * BN + (int)rank * (BN / CTAS);
        for (int kb = k_first; kb < k_last; ++kb) {
          const int s = (int)(issued % S::kStages);
          if (!mbar_wait_all(&empty[s], ((uint32_t)(issued / S::kStages) & 1u) ^ 1u)) {
            if (one) atomicExch(a.error, kErrEmptyWait);
            failed = true;
            break;
          }
          if (one) {
            if (leader) mbar_expect_tx(&full[s], CTAS == 2 ? 2 * S::kStage : S::kB + a.box_m * 128);  // the stage's bytes of both CTAs
            unsigned char* st = tiles + s * S::kStage;
            const uint32_t bar = smem_u32(&full[s]) & kPeerMask;
            if (CTAS == 1) {
              tma_load_2d(st, &map_a, &full[s], kb * 64, m0);
              tma_load_2d(st + S::kA, &map_b, &full[s], kb * 64, n0);
            } else if (A_MN) {
#pragma unroll
              for (int i = 0; i < 2; ++i) tma_load_2d_pair(st + i * 8192, &map_a, bar, m0 + 64 * i, kb * 64);
            } else {
              tma_load_2d_pair(st, &map_a, bar, kb * 64, m0);
            }
            if (CTAS == 1) {
            } else if (B_MN) {
#pragma unroll
              for (int i = 0; i < BN / 128; ++i)
                tma_load_2d_pair(st + S::kA + i * 8192, &map_b, bar, n0 + 64 * i, (a.second && kb >= a.second ? kb - a.second : kb) * 64);
            } else {
              tma_load_2d_pair(st + S::kA, &map_b, bar, kb * 64, n0);
            }
          }
          __syncwarp();
          ++issued;
        }
      }
    }
    // every stage this CTA filled has been consumed (released by the leader's MMAs) before exit
    for (int64_t j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
      if (!mbar_wait_all(&empty[j % S::kStages], (uint32_t)(j / S::kStages) & 1u) && one) atomicExch(a.error, kErrEmptyWait);
  } else if (warp == 1) {
    if (leader) {  // MMA issue: the leader only
      const bool one = elect_one();
      const uint32_t type = a.f16 ? 0u : 1u;
      const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                             ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);  // D float32, M = 128 or 256
      int64_t used = 0;
      int it = 0;  // accumulations so far
      bool failed = false;
      for (int u = first; u < a.units && !failed; u += step) {
        int split, mb, sg;
        unit_at<kRows>(a, u, split, mb, sg);
        const int k_first = (int)((int64_t)a.num_k * split / a.splits), k_last = (int)((int64_t)a.num_k * (split + 1) / a.splits);
        for (int nb = sg * a.seg; nb < min((sg + 1) * a.seg, n_blocks) && !failed; ++nb) {
          for (int k0 = k_first; k0 < k_last && !failed; k0 += a.chunk, ++it) {
            const int b = it & 1;
            if (!mbar_wait_all(&acc_empty[b], ((uint32_t)(it >> 1) & 1u) ^ 1u)) {
              if (one) atomicExch(a.error, kErrAccWait);
              failed = true;
              break;
            }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(b * 256);
            for (int kb = k0; kb < min(k0 + a.chunk, k_last); ++kb) {
              const int s = (int)(used % S::kStages);
              if (!mbar_wait_all(&full[s], (uint32_t)(used / S::kStages) & 1u)) {
                if (one) atomicExch(a.error, kErrFullWait);
                failed = true;
                break;
              }
              tc_fence_after();
              const unsigned char* st = tiles + s * S::kStage;
              const uint64_t ad = A_MN ? umma_desc_mn128(st) : umma_desc_sw128(st);
              const uint64_t bd = B_MN ? umma_desc_mn128(st + S::kA) : umma_desc_sw128(st + S::kA);
              if (one) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {  // 16 of K per MMA: 32 bytes of each row, or two groups of eight rows
                  const uint64_t a_desc = ad + (A_MN ? 128ull : 2ull) * kk, b_desc = bd + (B_MN ? 128ull : 2ull) * kk;
                  if (CTAS == 2)
                    umma_f16_pair(d, a_desc, b_desc, idesc, (kb > k0 || kk > 0) ? 1u : 0u);
                  else
                    umma_f16(d, a_desc, b_desc, idesc, (kb > k0 || kk > 0) ? 1u : 0u);
                }
                commit<CTAS>(&empty[s]);  // the stage is free again in both CTAs
              }
              __syncwarp();
              ++used;
            }
            if (one) commit<CTAS>(&acc_full[b]);  // both CTAs' accumulator halves complete
            __syncwarp();
            last_it[b] = it;
          }
        }
      }
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2;
    unsigned char* turn = turns + (warp - 2) * kOutBytes;
    const uint32_t buffer = smem_u32(turn);
    constexpr int kMine = S::kMine;  // columns of this warp
    float* bias = biases + (warp - 2) * kMine;
    int it = 0, next_nb = -1;
    float next_bias[(kMine + 31) / 32] = {};
    bool failed = false;
    for (int u = first; u < a.units; u += step) {
      int split, mb, sg;
      unit_at<kRows>(a, u, split, mb, sg);
      const int k_first = (int)((int64_t)a.num_k * split / a.splits), k_last = (int)((int64_t)a.num_k * (split + 1) / a.splits);
      const int m = mb * kRows + (int)rank * 128 + quad * 32 + lane;
      float top = -INFINITY, sum = 0.0f;  // kPartials: sum 2^top
      int64_t y = -1;                     // column of the row's target
      float weight = 0.0f, share = 0.0f, factor = 1.0f;  // of a gradient: softmax times weight is 2^(l - top) share
      if (EPI != kProduct && m < a.M) {
        const int64_t t = target_of(a.targets, m);
        y = t - a.first;
        if (EPI != kPartials) {
          const float2 z = __ldg(a.sums + m);
          top = z.x;
          weight = a.unit;
          if (a.row_grad) {
            const float most = __ldg(a.top_grad);
            const float own = __ldg(a.row_grad + m);
            weight *= most > 0.0f ? own / most : own * 0.0f;  // zeros but for what is not finite, which stays NaN
          }
          if (t < 0 || t >= a.categories) weight = __uint_as_float(0x7FC00000u);
          if (z.y == 0.0f || t == a.targets.ignored) weight = 0.0f;
          share = weight / z.y;  // the sum beside its maximum: their logarithm would be rounded at the size of the logits
        }
      }
      if (EPI == kProduct && a.scaled) factor = factor_of(a.factor) / a.unit;
      // what becomes of 32 sums of this thread's row, from column n on (called by whole warps)
      const auto finish = [&](float (&v)[32], int n) {
        const int live = min(32, a.N - n);
        if (a.beside ? n >= a.beside : live <= 0) return;
        if (EPI != kProduct) {
          if (a.bias) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 w = *reinterpret_cast<const float4*>(bias + n % kMine + 4 * i);
              add2(v[4 * i], v[4 * i + 1], w.x, w.y);
              add2(v[4 * i + 2], v[4 * i + 3], w.z, w.w);
            }
          }
          if (live < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = j < live ? v[j] : -INFINITY;
          }
        }
        if (EPI == kPartials) {
          const bool mine = y >= n && y < n + live;
          if (__any_sync(0xffffffffu, (int)mine)) {
            float z = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) z = y - n == j ? v[j] : z;
            if (mine) a.target_logit[m] = z;
          }
          float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int j = 4; j < 32; ++j) most[j & 3] = fmaxf(most[j & 3], v[j]);
          const float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * kLog2E;
          if (now > top) {
            sum *= top == -INFINITY ? 0.0f : exp2_fast(top - now);
            top = now;
          }
          const float base = top == -INFINITY ? 0.0f : -top;
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float e0, e1;
            fma2(v[j], v[j + 1], kLog2E, base, e0, e1);
            add2(s[j & 2], s[(j & 2) + 1], exp2_fast(e0), exp2_fast(e1));
          }
          sum += (s[0] + s[1]) + (s[2] + s[3]);
        } else if (EPI == kGradient || EPI == kGradientSums) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            fma2(v[j], v[j + 1], kLog2E, -top, v[j], v[j + 1]);
            v[j] = exp2_fast(v[j]);
            v[j + 1] = exp2_fast(v[j + 1]);
            mul2(v[j], v[j + 1], share);
          }
          // asked of the whole warp: the selections are 64 instructions that most pieces of a row need not make
          const int hit = y >= n && y < n + live ? (int)(y - n) : -1;
          if (__any_sync(0xffffffffu, (int)(hit >= 0))) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = hit == j ? v[j] - weight : v[j];
          }
          if (__any_sync(0xffffffffu, (int)(weight == 0.0f))) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = weight == 0.0f ? 0.0f : v[j];  // a row that does not count, whatever it holds
          }
          __syncwarp();
          if (EPI == kGradientSums) {
            const float s = column_sums(v);
            if (m - lane < a.M && lane < live) a.bias_part[(int64_t)(m >> 5) * a.bias_ld + n + lane] = s;
          }
          if (m < (a.second ? a.second : a.M)) {  // those behind the last row are zeros
            unsigned char* out = (unsigned char*)a.out + 2 * ((int64_t)m * a.out_ld + n);  // whole 32 columns: g_ld has room
            uint4 w[4];
            pack_row<4>(v, a.out_dtype, w);
            store_sector(out, w[0], w[1]);
            store_sector(out + 32, w[2], w[3]);
            if (a.second || a.beside) {
              less_row(v, a.out_dtype, w);
              pack_row<4>(v, a.out_dtype, w);
              out += 2 * (a.second * a.out_ld + a.beside);
              store_sector(out, w[0], w[1]);
              store_sector(out + 32, w[2], w[3]);
            }
          }
        } else if (a.tma_store) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) mul2(v[j], v[j + 1], factor);
          if (m - lane >= a.M) return;
          if (a.out_dtype == TTHRML_DT_F32) {
            sent_rows_read<0>();
            uint4 w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                __float_as_uint(v[4 * i + 3]));
            stage_row(buffer, w);
            send_rows(&map_out, buffer, n, m - lane, split, a.accumulate != 0);
          } else {  // 64 columns at a time
            uint4 w[4];
            pack_row<4>(v, a.out_dtype, w);
            const bool second = (n & 32) != 0;
            if (!second) sent_rows_read<0>();
            stage_row(buffer, w, second ? 4u : 0u);
            if (second || n + 32 >= a.N) send_rows(&map_out, buffer, n & ~63, m - lane, split);
          }
        } else {
          if (a.carry && m < a.M) {  // a row per lane: a long main loop hides it
            const float4* old = reinterpret_cast<const float4*>(a.carry + (int64_t)m * a.carry_ld + n);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 c = __ldcg(old + i);
              add2(v[4 * i], v[4 * i + 1], c.x, c.y);
              add2(v[4 * i + 2], v[4 * i + 3], c.z, c.w);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) mul2(v[j], v[j + 1], factor);
          if (a.align == 16 && a.out_dtype != TTHRML_DT_F32 && live == 32) {
            uint4 w[4];
            pack_row<4>(v, a.out_dtype, w);
            store_rows64(w, buffer, (unsigned char*)a.out + 2 * n, 2 * a.out_ld, m - lane, a.M);
          } else {
            store_values(v, a.out_dtype, turn, (unsigned char*)a.out, a.out_ld, n, m - lane, a.M, live, a.align);
          }
        }
      };
      for (int nb = sg * a.seg; nb < min((sg + 1) * a.seg, n_blocks); ++nb) {
        if (EPI != kProduct && a.bias) {  // each warp keeps its own columns' biases: no barrier of all of them
          const auto fetch = [&](int block) {
#pragma unroll
            for (int i = 0; i < kMine / 32; ++i) {
              const int n = block * BN + part * kMine + 32 * i + lane;
              next_bias[i] = n < a.N ? __ldg(a.bias + n) : 0.0f;
            }
          };
          if (next_nb != nb) fetch(nb);
          __syncwarp();  // the lanes have read those of the tile before
#pragma unroll
          for (int i = 0; i < kMine / 32; ++i) bias[32 * i + lane] = next_bias[i];
          __syncwarp();
          next_nb = nb + 1;  // the next tile's are on their way meanwhile: of this unit, or of the next one
          if (next_nb >= min((sg + 1) * a.seg, n_blocks) && u + step < a.units) {
            int next_split, next_mb, next_sg;
            unit_at<kRows>(a, u + step, next_split, next_mb, next_sg);
            next_nb = next_sg * a.seg;
          }
          fetch(next_nb);
        }
        if constexpr (kChunked) {
          float acc[kMine];
#pragma unroll
          for (int j = 0; j < kMine; ++j) acc[j] = 0.0f;
          for (int k0 = k_first; k0 < k_last && !failed; k0 += a.chunk, ++it) {
            const int b = it & 1;
            if (!mbar_wait_warp(&acc_full[b], (uint32_t)(it >> 1) & 1u)) {
              if (lane == 0) atomicExch(a.error, kErrAccWait);
              failed = true;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < kMine / 16; ++q) {
              float v[16];
              tmem_load16(tmem + (uint32_t)(b * 256) + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * kMine + q * 16), v);
#pragma unroll
              for (int j = 0; j < 16; j += 2) add2(acc[q * 16 + j], acc[q * 16 + j + 1], v[j], v[j + 1]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(&acc_empty[b]);
          }
          if (failed) break;
#pragma unroll
          for (int q = 0; q < kMine / 32; ++q) {
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = acc[q * 32 + j];
            finish(v, nb * BN + part * kMine + q * 32);
          }
        } else {
          if (!failed && !mbar_wait_warp(&acc_full[it & 1], (uint32_t)(it >> 1) & 1u)) {
            if (lane == 0) atomicExch(a.error, kErrAccWait);
            failed = true;
          }
          if (failed) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = part * kMine; c < (part + 1) * kMine; c += 32) {
            float v[32];
            tmem_load32(tmem + (uint32_t)((it & 1) * 256) + ((uint32_t)(quad * 32) << 16) + (uint32_t)c, v);
            finish(v, nb * BN + c);
            __syncwarp();  // the next TMEM load is a warp's
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(&acc_empty[it & 1]);
          ++it;
        }
      }
      if (EPI == kPartials && m < a.M) a.part[(int64_t)m * a.slots + S::kParts * sg + part] = make_float2(top, sum);
    }
    if (EPI == kProduct) sent_rows_done();
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
  if (warp == 1) {
    if (CTAS == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Joins the partial sums of a row (a warp per row) into one and the row's loss, in 64 bits from there on; the last block adds the losses, in an
// order that does not depend on which block is the last.
struct LossArgs {
  const float2* part;
  const float* target_logit;
  RowTargets targets;
  int64_t rows, categories;
  int32_t slots, reduction;  // 0: none, 1: mean over the rows that count, 2: sum
  float2* sums;              // [rows]
  float* loss;               // [rows]
  float *total, *inv_count;  // the reduced loss, and 1 / the rows that count (1 at least) or 1
  uint32_t* counter;
};
__global__ void __launch_bounds__(256) k_xent_loss(const LossArgs a) {
  __shared__ double sums[8];
  __shared__ int64_t counts[8];
  __shared__ bool last;
  let_next_kernel_start();
  wait_for_previous_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + warp;
  if (row < a.rows) {
    float m = -INFINITY, s = 0.0f;
    const float2* p = a.part + row * a.slots;
    for (int i = lane; i < a.slots; i += 32) {
      const float2 v = __ldcg(p + i);
      join(m, s, v.x, v.y);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      if (lane & o) {  // both lanes of a pair join in the same order
        float m1 = m2, s1 = s2;
        join(m1, s1, m, s);
        m = m1, s = s1;
      } else {
        join(m, s, m2, s2);
      }
    }
    if (lane == 0) {
      const int64_t y = target_of(a.targets, row);
      float loss = 0.0f;
      if (y != a.targets.ignored) {
        if (y < 0 || y >= a.categories)
          loss = __uint_as_float(0x7FC00000u);
        else
          loss = s == 0.0f ? INFINITY  // no category is possible
                           : (float)(((double)m + log2((double)s)) * (1.0 / (double)kLog2E) - (double)__ldcg(a.target_logit + row));
      }
      a.sums[row] = make_float2(m, s);
      a.loss[row] = loss;
    }
  }
  if (a.reduction == 0) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1u;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0;
  int64_t count = 0;
  for (int64_t i = threadIdx.x; i < a.rows; i += 256) {
    sum += (double)__ldcg(a.loss + i);
    count += target_of(a.targets, i) != a.targets.ignored;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) sums[warp] = sum, counts[warp] = count;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum += sums[i], count += counts[i];
    const double n = a.reduction == 1 ? (double)(count > 0 ? count : 1) : 1.0;
    *a.total = (float)(sum / n);
    *a.inv_count = (float)(1.0 / n);
  }
}

// The largest finite magnitude of the weights of the rows that count (one that is not stays with its own row); one block.
__global__ void __launch_bounds__(1024) k_xent_top(const float* grad, RowTargets targets, int64_t rows, float* top) {
  __shared__ float part[32];
  let_next_kernel_start();
  wait_for_previous_kernel();
  float most = 0.0f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024)
    if (target_of(targets, i) != targets.ignored) {
      const float size = fabsf(__ldg(grad + i));
      if (size < INFINITY) most = fmaxf(most, size);
    }
  for (int o = 16; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x < 32) {
    most = part[threadIdx.x];
    for (int o = 16; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (threadIdx.x == 0) *top = most;
  }
}

// out[r][c] = factor * sum of planes[i][r][c], in the order of the planes.
struct JoinArgs {
  const float* planes;
  int64_t plane, ld, rows, cols;
  int64_t second;  // rows further lies another part of each row's sum; 0: none
  int32_t n;
  void* out;
  int64_t out_ld;
  int32_t out_dtype;
  const float* factor[2];
  float unit;
};
__device__ __forceinline__ void join_rows(const JoinArgs& a, int64_t block, int64_t blocks) {
  const float factor = factor_of(a.factor) / a.unit;
  const int64_t quads = (a.cols + 3) / 4, all = a.rows * quads;
  for (int64_t i = block * 256 + threadIdx.x; i < all; i += blocks * 256) {
    const int64_t r = i / quads, c = (i - r * quads) * 4;
    const float* p = a.planes + r * a.ld + c;
    float4 s = __ldcg(reinterpret_cast<const float4*>(p));
    const int parts = a.second ? 2 * a.n : a.n;
    for (int k = 1; k < parts; ++k) {
      const float* q = k < a.n ? p + k * a.plane : p + (k - a.n) * a.plane + a.second * a.ld;
      const float4 t = __ldcg(reinterpret_cast<const float4*>(q));
      s.x += t.x, s.y += t.y, s.z += t.z, s.w += t.w;
    }
    const float v[4] = {s.x * factor, s.y * factor, s.z * factor, s.w * factor};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j >= a.cols) break;
      const int64_t at = r * a.out_ld + c + j;
      if (a.out_dtype == TTHRML_DT_F32)
        reinterpret_cast<float*>(a.out)[at] = v[j];
      else if (a.out_dtype == TTHRML_DT_BF16)
        reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v[j]);
      else
        reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v[j]);
    }
  }
}

// db[n] = factor * sum over the groups of 32 rows, in their order and in 64 bits (there may be half a million); eight threads share
// a column.
struct BiasArgs {
  const float* part;
  int64_t groups, ld, n;
  float* db;
  const float* factor[2];
  float unit;
};
__device__ __forceinline__ void bias_sums(const BiasArgs& a, int64_t block) {
  __shared__ double sums[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = block * 32 + lane;
  double s = 0.0;
  if (c < a.n) {
#pragma unroll 4
    for (int64_t g = warp; g < a.groups; g += 8) s += (double)__ldcg(a.part + g * a.ld + c);
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < a.n) {
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
    a.db[c] = (float)(s * (double)(factor_of(a.factor) / a.unit));
  }
}

// What the products of a piece leave to add up: planes of dx, planes of dw, the sums for db; a range of blocks each.
struct FinishArgs {
  JoinArgs x, w;
  BiasArgs b;
  int32_t x_blocks, w_blocks, b_blocks;
};
__global__ void __launch_bounds__(256) k_xent_finish(const __grid_constant__ FinishArgs a) {
  let_next_kernel_start();
  wait_for_previous_kernel();
  int64_t block = blockIdx.x;
  if (block < a.x_blocks) {
    join_rows(a.x, block, a.x_blocks);
  } else if ((block -= a.x_blocks) < a.w_blocks) {
    join_rows(a.w, block, a.w_blocks);
  } else {
    bias_sums(a.b, block - a.w_blocks);
  }
}

// Tensor map of a 16-bit matrix [rows][cols] with rows ld elements apart, in boxes of 64 columns x box_rows, 128-byte swizzle.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows, bool f16) {
  EncodeTiledFn fn;
  int rc = encode_fn(&fn);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64u, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for a %lld x %lld 16-bit matrix", (int)r, (long long)rows, (long long)cols);
    return TTHRML_ERR_CUDA;
  }
  return TTHRML_OK;
}

constexpr int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

template <int EPI, bool A_MN, bool B_MN, int BN, int CTAS, bool BRIEF>
int launch_xent(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const XentArgs& a, cudaStream_t st) {
  const void* fn = (const void*)k_xent<EPI, A_MN, B_MN, BN, CTAS, BRIEF>;
  constexpr int kThreads = XentShape<EPI, BN, CTAS, BRIEF>::kThreads, kSmem = XentShape<EPI, BN, CTAS, BRIEF>::kSmem;
  ClusterFit fit;
  const int rc = cluster_fit(fn, CTAS, kThreads, kSmem, &fit);
  if (rc) return rc;
  const int64_t clusters = a.units < fit.clusters ? a.units : fit.clusters;
  void* params[4] = {(void*)&ma, (void*)&mb, (void*)&mo, (void*)&a};
  return launch_clusters(fn, (unsigned)(CTAS * clusters), CTAS, kThreads, kSmem, params, st, "k_xent launch", true);
}
template <int EPI, int CTAS, bool BRIEF>
int launch_logits(int bn, const CUtensorMap& ma, const CUtensorMap& mb, const XentArgs& a, cudaStream_t st) {
  if (bn == 64) return launch_xent<EPI, false, false, 64, CTAS, BRIEF>(ma, mb, ma, a, st);
  if (bn == 128) return launch_xent<EPI, false, false, 128, CTAS, BRIEF>(ma, mb, ma, a, st);
  return launch_xent<EPI, false, false, 256, CTAS, BRIEF>(ma, mb, ma, a, st);
}
template <int EPI>
int launch_logits(int ctas, int bn, bool brief, const CUtensorMap& ma, const CUtensorMap& mb, XentArgs a, cudaStream_t st) {
  if (brief) {
    a.chunk = a.num_k;
    return ctas == 1 ? launch_logits<EPI, 1, true>(bn, ma, mb, a, st) : launch_logits<EPI, 2, true>(bn, ma, mb, a, st);
  }
  return ctas == 1 ? launch_logits<EPI, 1, false>(bn, ma, mb, a, st) : launch_logits<EPI, 2, false>(bn, ma, mb, a, st);
}

// How many pairs of CTAs work at once (every form of the kernel fills an SM).
int resident_pairs(int64_t* out) {
  ClusterFit fit;
  const int rc = cluster_fit((const void*)k_xent<kProduct, false, true, 256, 2, false>, 2,
                             XentShape<kProduct, 256, 2, false>::kThreads, XentShape<kProduct, 256, 2, false>::kSmem, &fit);
  *out = fit.clusters;
  return rc;
}
// CTAs per tile of logits, and the widest tile that still gives every cluster work.
int tile_ctas(int64_t rows) { return rows <= 128 ? 1 : 2; }
int box_rows(int64_t rows) { return rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 64 ? 64 : 128)); }
int tile_width(int64_t rows, int64_t n, int64_t pairs) {
  const int64_t ctas = tile_ctas(rows), m_blocks = up(rows, 128 * ctas) / (128 * ctas), at_once = pairs * 2 / ctas;
  for (int bn = 256; bn > 64; bn /= 2)
    if (n > bn / 2 && m_blocks * (up(n, bn) / bn) >= at_once) return bn;
  return 64;
}
// Tiles along N per unit: as few rounds of units as possible, then as few partial sums.
int tiles_per_unit(int64_t m_blocks, int64_t n_blocks, int64_t pairs) {
  int64_t best = INT64_MAX, seg = 1;
  for (int64_t s = 1; s <= n_blocks && s <= 128; ++s) {
    const int64_t units = m_blocks * ((n_blocks + s - 1) / s), cost = (units + pairs - 1) / pairs * s;
    if (cost <= best) best = cost, seg = s;
  }
  return (int)seg;
}
// Shares of a product's sum: as many as give every pair a tile, of at least four blocks of 64.
int64_t shares(int64_t m, int64_t n, int64_t k, int64_t pairs) {
  const int64_t tiles = (up(m, 256) / 256) * (up(n, 256) / 256), most = std::max<int64_t>(1, up(k, 64) / 64 / 4);
  return std::max<int64_t>(1, std::min(pairs / tiles, most));
}

struct ForwardPlan {
  int bn, seg, segments, slots;
  int64_t logits, counter, bytes;  // places in the workspace behind the partial sums
};
int plan_forward(int64_t rows, int64_t categories, int64_t cols, ForwardPlan* p) {
  int64_t pairs;
  const int rc = resident_pairs(&pairs);
  if (rc) return rc;
  p->bn = tile_width(rows, categories, pairs);
  const int64_t n_blocks = up(categories, p->bn) / p->bn;
  const int64_t ctas = tile_ctas(rows);
  p->seg = tiles_per_unit(up(rows, 128 * ctas) / (128 * ctas), n_blocks, pairs * 2 / ctas);
  p->segments = (int)((n_blocks + p->seg - 1) / p->seg);
  p->slots = parts_of(one_chunk(rows, categories, cols), p->bn) * p->segments;
  p->logits = up(rows * p->slots * 8, 16);
  p->counter = p->logits + up(rows * 4, 16);
  p->bytes = p->counter + 16;
  return TTHRML_OK;
}

struct BackwardPlan {
  int64_t piece, pieces, g_ld, plane_ld, dx_shares, dw_shares;
  int64_t second, beside;  // the row or the column where the second pieces begin (0: none)
  int64_t g_rows, g_cols;  // of g with them, of a piece
  bool dx_planes, dw_planes;
  int64_t bias, top, dx, dw, bytes;  // places in the workspace behind g
};
int plan_backward(int64_t rows, int64_t categories, int64_t cols, bool want_x, bool want_w, bool want_b, BackwardPlan* p) {
  int64_t pairs;
  const int rc = resident_pairs(&pairs);
  if (rc) return rc;
  p->beside = categories <= kFewCategories ? kFewCategories : 0;
  p->second = rows <= kFewRows && !p->beside ? up(rows, 64) : 0;
  p->g_rows = p->second ? 2 * p->second : rows;
  const int64_t most = std::max<int64_t>(256, kPieceBytes / 2 / p->g_rows / 256 * 256);
  p->pieces = (categories + most - 1) / most;
  p->piece = up((categories + p->pieces - 1) / p->pieces, 256);
  p->pieces = (categories + p->piece - 1) / p->piece;
  const int64_t width = std::min(p->piece, categories);
  p->g_cols = p->beside ? 2 * p->beside : width;
  p->g_ld = up(p->g_cols, 64);
  p->plane_ld = up(cols, 32);
  p->dx_shares = want_x ? shares(p->g_rows, cols, p->g_cols, pairs) : 0;
  p->dw_shares = want_w ? shares(p->g_cols, cols, p->g_rows, pairs) : 0;
  p->dx_planes = want_x && (p->dx_shares > 1 || p->pieces > 1 || p->second);
  p->dw_planes = want_w && (p->dw_shares > 1 || p->beside);
  p->bias = up(p->g_rows * p->g_ld * 2, 16);
  p->top = p->bias + (want_b ? up(rows, 32) / 32 * p->g_ld * 4 : 0);
  p->dx = p->top + 16;
  p->dw = p->dx + (p->dx_planes ? p->dx_shares * p->g_rows * p->plane_ld * 4 : 0);
  p->bytes = p->dw + (p->dw_planes ? p->dw_shares * p->g_cols * p->plane_ld * 4 : 0);
  return TTHRML_OK;
}

int check_problem(const char* what, const tthrml_xent* p) {
  if (!p || !p->x || !p->w || !p->targets) {
    set_error("%s: NULL argument", what);
    return TTHRML_ERR_ARG;
  }
  if (p->dtype != TTHRML_DT_BF16 && p->dtype != TTHRML_DT_F16) {
    set_error("%s: x and weights must be bfloat16 or float16 (got code %d)", what, (int)p->dtype);
    return TTHRML_ERR_ARG;
  }
  if (p->rows < 1 || p->categories < 1 || p->cols < 1 || p->rows > TTHRML_XENT_MAX_ROWS ||
      p->categories > TTHRML_XENT_MAX_CATEGORIES || p->cols > TTHRML_XENT_MAX_COLS) {
    set_error("%s: sizes out of range (%lld rows of %lld columns, %lld categories)", what, (long long)p->rows,
              (long long)p->cols, (long long)p->categories);
    return TTHRML_ERR_ARG;
  }
  if ((uintptr_t)p->x % 16 || (uintptr_t)p->w % 16 || p->x_ld % 8 || p->w_ld % 8 || p->x_ld < p->cols || p->w_ld < p->cols ||
      (uintptr_t)p->targets % (p->wide_targets ? 8 : 4) || (p->bias && (uintptr_t)p->bias % 4)) {
    set_error("%s: x and weights must be 16-byte aligned with pitches that are multiples of 8 elements and not below the "
              "columns (got pitches %lld, %lld)", what, (long long)p->x_ld, (long long)p->w_ld);
    return TTHRML_ERR_ARG;
  }
  return TTHRML_OK;
}

// One product of the backward pass, [m][k] x [k][n], into out (scaled) or planes.
template <bool A_MN>
int product(const CUtensorMap& ma, const CUtensorMap& mb, XentArgs a, int64_t m, int64_t n, int64_t k, int64_t n_shares,
            int64_t pairs, cudaStream_t st) {
  a.M = (int32_t)m;
  a.N = (int32_t)n;
  a.num_k = (int32_t)(up(k, 64) / 64);
  a.seg = 1;
  a.segments = (int32_t)(up(n, 256) / 256);
  a.splits = (int32_t)n_shares;
  const int64_t m_blocks = up(m, 256) / 256;
  a.units = (int32_t)(m_blocks * a.segments * n_shares);
  int64_t g = 1;  // about square rectangles of the tiles in flight
  while ((g + 1) * (g + 1) <= pairs) ++g;
  a.group = (int32_t)std::min(g, m_blocks);
  a.chunk = a.num_k;
  CUtensorMap mo = ma;  // never used where the rows are not aligned
  // Bulk stores are the quicker way out of short sums, but queue behind the loads of long ones, as in the 4-bit product.
  a.tma_store = (!a.scaled || (a.num_k <= 8 && !a.carry)) && make_out_map(&mo, a.out, m, n, a.out_ld, a.out_dtype, n_shares, m * a.out_ld);
  if (!a.scaled && !a.tma_store) {
    set_error("planes of %lld x %lld sums take no tensor map", (long long)m, (long long)n);
    return TTHRML_ERR_CUDA;
  }
  return launch_xent<kProduct, A_MN, true, 256, 2, false>(ma, mb, mo, a, st);
}
void join_later(JoinArgs& j, int32_t& blocks, const float* planes, int64_t plane, int64_t ld, int64_t rows, int64_t cols,
                int64_t second, int64_t n, const XentArgs& a, void* out, int64_t out_ld, int32_t out_dtype) {
  j = {planes, plane, ld, rows, cols, second, (int32_t)n, out, out_ld, out_dtype, {a.factor[0], a.factor[1]}, a.unit};
  blocks = (int32_t)std::min<int64_t>((rows * ((cols + 3) / 4) + 255) / 256, 148 * 8);
}

}  // namespace
}  // namespace tthrml

extern "C" int64_t tthrml_xent_forward_workspace(int64_t rows, int64_t categories, int64_t cols) {
  using namespace tthrml;
  if (rows < 1 || categories < 1 || cols < 1 || rows > TTHRML_XENT_MAX_ROWS || categories > TTHRML_XENT_MAX_CATEGORIES ||
      cols > TTHRML_XENT_MAX_COLS)
    return 0;
  ForwardPlan p;
  const int rc = plan_forward(rows, categories, cols, &p);
  return rc ? rc : p.bytes;
}

extern "C" int tthrml_xent_forward(const tthrml_xent* p, float* sums, float* row_loss, float* loss, float* inv_count,
                                   int32_t reduction, void* workspace, int64_t workspace_bytes, int32_t* error, void* stream) {
  using namespace tthrml;
  int rc = check_problem("tthrml_xent_forward", p);
  if (rc) return rc;
  if (!sums || (uintptr_t)sums % 8 || !row_loss || !workspace || !error || reduction < 0 || reduction > 2 || (reduction && (!loss || !inv_count))) {
    set_error("tthrml_xent_forward: NULL argument, sums not 8-byte aligned or unknown reduction %d", (int)reduction);
    return TTHRML_ERR_ARG;
  }
  ForwardPlan f;
  rc = plan_forward(p->rows, p->categories, p->cols, &f);
  if (rc) return rc;
  if ((uintptr_t)workspace % 16 || workspace_bytes < f.bytes) {
    set_error("tthrml_xent_forward: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)f.bytes,
              (long long)workspace_bytes);
    return TTHRML_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = p->dtype == TTHRML_DT_F16;
  unsigned char* ws = (unsigned char*)workspace;
  const int ctas = tile_ctas(p->rows);
  CUtensorMap ma, mb;
  rc = make_map(&ma, p->x, p->rows, p->cols, p->x_ld, (uint32_t)box_rows(p->rows), f16);
  if (rc == TTHRML_OK) rc = make_map(&mb, p->w, p->categories, p->cols, p->w_ld, (uint32_t)(f.bn / ctas), f16);
  if (rc) return rc;
  XentArgs a = {};
  a.M = (int32_t)p->rows;
  a.N = (int32_t)p->categories;
  a.num_k = (int32_t)(up(p->cols, 64) / 64);
  a.f16 = f16;
  a.box_m = box_rows(p->rows);
  a.seg = f.seg;
  a.segments = f.segments;
  a.splits = 1;
  const int64_t m_blocks = up(p->rows, 128 * ctas) / (128 * ctas), g = ((int64_t)32 << 20) / (512 * p->cols);
  a.units = (int32_t)(m_blocks * f.segments);
  a.group = (int32_t)std::max<int64_t>(1, std::min(g, m_blocks));  // raster groups of about 32 MiB of A panels
  a.bias = p->bias;
  a.categories = p->categories;
  a.targets = {p->targets, p->wide_targets, p->ignored};
  a.part = (float2*)ws;
  a.slots = f.slots;
  a.target_logit = (float*)(ws + f.logits);
  a.counter = (uint32_t*)(ws + f.counter);
  a.error = error;
  a.chunk = chunk_of(p->rows, p->categories);
  rc = launch_logits<kPartials>(ctas, f.bn, one_chunk(p->rows, p->categories, p->cols), ma, mb, a, st);
  if (rc) return rc;
  LossArgs l = {a.part, a.target_logit, a.targets, p->rows, p->categories, a.slots, reduction, (float2*)sums, row_loss, loss, inv_count,
                a.counter};
  void* params[1] = {(void*)&l};
  return launch_clusters((const void*)k_xent_loss, (unsigned)((p->rows + 7) / 8), 1, 256, 0, params, st, "k_xent_loss launch",
                         true);
}

extern "C" int64_t tthrml_xent_backward_workspace(int64_t rows, int64_t categories, int64_t cols, int32_t dx, int32_t dw,
                                                  int32_t db) {
  using namespace tthrml;
  if (rows < 1 || categories < 1 || cols < 1 || rows > TTHRML_XENT_MAX_ROWS || categories > TTHRML_XENT_MAX_CATEGORIES ||
      cols > TTHRML_XENT_MAX_COLS)
    return 0;
  BackwardPlan p;
  const int rc = plan_backward(rows, categories, cols, dx != 0, dw != 0, db != 0, &p);
  return rc ? rc : p.bytes;
}

extern "C" int tthrml_xent_backward(const tthrml_xent* p, const float* sums, const float* grad, int32_t grad_per_row,
                                    const float* inv_count, void* dx, int64_t dx_ld, void* dw, int64_t dw_ld,
                                    int32_t grad_dtype, float* db, void* workspace, int64_t workspace_bytes, int32_t* error,
                                    void* stream) {
  using namespace tthrml;
  int rc = check_problem("tthrml_xent_backward", p);
  if (rc) return rc;
  if (!sums || (uintptr_t)sums % 8 || !grad || !workspace || !error || (dx && dx_ld < p->cols) || (dw && dw_ld < p->cols)) {
    set_error("tthrml_xent_backward: NULL argument, sums not 8-byte aligned, or gradients whose rows overlap");
    return TTHRML_ERR_ARG;
  }
  if (grad_dtype == TTHRML_DT_I8 || dtype_bytes(grad_dtype) == 0) {
    set_error("tthrml_xent_backward: gradients must be float32, bfloat16 or float16 (got code %d)", (int)grad_dtype);
    return TTHRML_ERR_ARG;
  }
  if (!dx && !dw && !db) return TTHRML_OK;
  BackwardPlan f;
  rc = plan_backward(p->rows, p->categories, p->cols, dx, dw, db, &f);
  int64_t pairs;
  if (rc == TTHRML_OK) rc = resident_pairs(&pairs);
  if (rc) return rc;
  if ((uintptr_t)workspace % 32 || workspace_bytes < f.bytes) {
    set_error("tthrml_xent_backward: needs a 32-byte aligned workspace of %lld bytes (got %lld)", (long long)f.bytes,
              (long long)workspace_bytes);
    return TTHRML_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = p->dtype == TTHRML_DT_F16;
  unsigned char* ws = (unsigned char*)workspace;
  float* top = (float*)(ws + f.top);
  XentArgs base = {};
  base.f16 = f16;
  base.box_m = box_rows(p->rows);
  base.unit = f16 ? 16384.0f : 1.0f;
  base.categories = p->categories;
  base.targets = {p->targets, p->wide_targets, p->ignored};
  base.sums = (const float2*)sums;
  base.error = error;
  base.factor[0] = grad_per_row ? top : grad;
  base.factor[1] = inv_count;
  if (grad_per_row) {
    base.row_grad = grad;
    base.top_grad = top;
    void* params[4] = {(void*)&grad, (void*)&base.targets, (void*)&p->rows, (void*)&top};
    rc = launch_clusters((const void*)k_xent_top, 1, 1, 1024, 0, params, st, "k_xent_top launch", true);
    if (rc) return rc;
  }
  const int64_t bytes = dtype_bytes(grad_dtype);
  auto alignment = [&](const void* out, int64_t ld) {
    const uint64_t v = (uint64_t)(uintptr_t)out | (uint64_t)(ld * bytes);
    return v % 16 == 0 ? 16 : (v % 8 == 0 ? 8 : (v % 4 == 0 ? 4 : 2));
  };
  CUtensorMap mx, mx_mn;
  rc = make_map(&mx, p->x, p->rows, p->cols, p->x_ld, (uint32_t)box_rows(p->rows), f16);
  if (rc == TTHRML_OK) rc = make_map(&mx_mn, p->x, p->rows, p->cols, p->x_ld, 64u, f16);
  for (int64_t i = 0; i < f.pieces && rc == TTHRML_OK; ++i) {
    const int64_t first = i * f.piece, width = std::min(f.piece, p->categories - first);
    const int64_t g_cols = f.beside ? f.g_cols : width;
    const char* w = (const char*)p->w + first * p->w_ld * 2;
    CUtensorMap mw, mw_mn, mg, mg_mn;
    FinishArgs finish = {};
    const int bn = tile_width(p->rows, width, pairs), ctas = tile_ctas(p->rows);
    rc = make_map(&mw, w, width, p->cols, p->w_ld, (uint32_t)(bn / ctas), f16);
    if (rc == TTHRML_OK) rc = make_map(&mw_mn, w, width, p->cols, p->w_ld, 64u, f16);
    if (rc == TTHRML_OK) rc = make_map(&mg, ws, f.g_rows, g_cols, f.g_ld, 128u, f16);
    if (rc == TTHRML_OK) rc = make_map(&mg_mn, ws, f.g_rows, g_cols, f.g_ld, 64u, f16);
    if (rc) return rc;
    XentArgs a = base;
    a.M = (int32_t)p->rows;
    a.N = (int32_t)width;
    a.num_k = (int32_t)(up(p->cols, 64) / 64);
    a.seg = 1;
    a.segments = (int32_t)(up(width, bn) / bn);
    a.splits = 1;
    const int64_t m_blocks = up(p->rows, 128 * ctas) / (128 * ctas);
    a.units = (int32_t)(m_blocks * a.segments);
    int64_t g = 1;
    while ((g + 1) * (g + 1) <= pairs) ++g;
    a.group = (int32_t)std::min(g, m_blocks);
    a.bias = p->bias ? p->bias + first : nullptr;
    a.first = first;
    a.bias_part = db ? (float*)(ws + f.bias) : nullptr;
    a.bias_ld = f.g_ld;
    a.chunk = chunk_of(p->rows, p->categories);  // as the forward pass: the sums belong to these logits
    a.second = (int32_t)f.second;
    a.beside = (int32_t)f.beside;
    a.out = ws;
    a.out_ld = f.g_ld;
    a.out_dtype = p->dtype;
    const bool brief = one_chunk(p->rows, p->categories, p->cols);
    rc = db ? launch_logits<kGradientSums>(ctas, bn, brief, mx, mw, a, st) : launch_logits<kGradient>(ctas, bn, brief, mx, mw, a, st);
    if (rc) return rc;
    if (dx) {
      XentArgs d = base;
      const bool ends = f.dx_planes && f.dx_shares == 1 && !f.second && i + 1 == f.pieces;  // takes the plane's sums along
      const bool planes = f.dx_planes && !ends;
      d.scaled = !planes;
      d.out = planes ? (void*)(ws + f.dx) : dx;
      d.out_ld = planes ? f.plane_ld : dx_ld;
      d.out_dtype = planes ? TTHRML_DT_F32 : grad_dtype;
      d.align = alignment(dx, dx_ld);
      d.accumulate = planes && i > 0;
      d.carry = ends ? (const float*)(ws + f.dx) : nullptr;
      d.carry_ld = f.plane_ld;
      d.second = (int32_t)(f.beside / 64);
      rc = product<false>(mg, mw_mn, d, f.g_rows, p->cols, g_cols, std::min(f.dx_shares, up(g_cols, 64) / 64), pairs, st);
      if (rc) return rc;
    }
    if (dw) {
      XentArgs d = base;
      char* out = (char*)dw + first * dw_ld * bytes;
      const bool planes = f.dw_planes;
      d.scaled = !planes;
      d.out = planes ? (void*)(ws + f.dw) : out;
      d.out_ld = planes ? f.plane_ld : dw_ld;
      d.out_dtype = planes ? TTHRML_DT_F32 : grad_dtype;
      d.align = alignment(out, dw_ld);
      d.second = (int32_t)(f.second / 64);
      rc = product<true>(mg_mn, mx_mn, d, g_cols, p->cols, f.g_rows, f.dw_shares, pairs, st);
      if (rc) return rc;
      if (planes)
        join_later(finish.w, finish.w_blocks, (const float*)(ws + f.dw), g_cols * f.plane_ld, f.plane_ld, width, p->cols, f.beside,
                   f.dw_shares, base, out, dw_ld, grad_dtype);
    }
    if (db) {
      finish.b = {a.bias_part, up(p->rows, 32) / 32, f.g_ld, width, db + first, {base.factor[0], base.factor[1]}, base.unit};
      finish.b_blocks = (int32_t)((width + 31) / 32);
    }
    if (dx && i + 1 == f.pieces && f.dx_planes && (f.dx_shares > 1 || f.second))
      join_later(finish.x, finish.x_blocks, (const float*)(ws + f.dx), f.g_rows * f.plane_ld, f.plane_ld, p->rows, p->cols, f.second,
                 f.dx_shares, base, dx, dx_ld, grad_dtype);
    const int64_t blocks = (int64_t)finish.x_blocks + finish.w_blocks + finish.b_blocks;
    if (blocks) {
      void* params[1] = {(void*)&finish};
      rc = launch_clusters((const void*)k_xent_finish, (unsigned)blocks, 1, 256, 0, params, st, "k_xent_finish launch", true);
    }
  }
  return rc;
}
