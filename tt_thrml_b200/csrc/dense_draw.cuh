// Draws of the dense (tensor-core) kernels' epilogues: spin and gaussian decisions of a 32-column chunk of fields,
// the near-threshold list and the raster order of the output tiles.  Shared by the bf16 and the 8-bit kernels.
#pragma once

#include "tc_common.cuh"

namespace tthrml {
namespace {

struct DenseArgs {
  const float* bias;       // [N] or NULL
  __nv_bfloat16* out;      // [M][pieces * N] new target state: bf16 pieces, value = sum over pieces
  float* out_f32;          // [M][N] same values in float32, or NULL
  int32_t pieces;          // 1: bf16 value; 2-3: successive bf16 remainders (3 is exact for float32)
  const float* variates;   // [variates_sweeps][N][M] (unit-major, chains innermost) or NULL
  int64_t variates_sweeps;
  int64_t M, N, K;
  int64_t row0;            // flat state row of target unit 0 (Philox counter)
  int64_t chain_offset;
  uint64_t seed;
  uint32_t sweep;
  int32_t family;          // TTHRML_SPIN or TTHRML_GAUSSIAN
  float precision;         // gaussian: sum of precision contributions (1 for unit variance)
  const tthrml_run_ctl* ctl;
  int* error;              // device word, set on a wait timeout
  uint32_t* ties;          // near-threshold spin decisions: [count, blocks done, dropped, 0, (m, n) x ties_cap]
  int64_t ties_cap;        // or NULL: decisions from the float32 field alone
  int32_t group;           // CTA-pair kernel: row blocks per raster group
};

// A spin decision whose float32 margin is this close to the threshold (in units of u * (1 + e^(-2 gamma))
// around 1, or of 2 gamma - logit in variates mode; |t - 1| ~ (1 - u) |2 gamma - logit u|) is decided
// again from the exact field.  The tensor cores' float32 accumulation of a K-term field can be off by
// ~1e-5 at K = 4096 with terms of size 0.01; a decision the float32 field gets wrong at a true margin
// beyond the 1e-5 band therefore shows a float32 margin below (error - 1e-5), which this bound catches
// for errors up to 2e-5.  The exact field is bias + sum_k A[m][k] B[n][k] in double (bf16 products are
// exact there).  The epilogue only records such decisions (a few in 10^5); k_dense_settle, launched
// next on the same stream, decides them again and overwrites their outputs.
constexpr float kNearTie = 1e-5f;
#ifndef TTHRML_DENSE_FAST_TRIG
#define TTHRML_DENSE_FAST_TRIG 1  // Box-Muller angle through the hardware sine / cosine (0: sincospif)
#endif
#ifndef TTHRML_DENSE_F32X2
#define TTHRML_DENSE_F32X2 1  // spin draws with packed f32x2 arithmetic (0: scalar)
#endif
#ifndef TTHRML_DENSE_SETTLE
#define TTHRML_DENSE_SETTLE 2  // 0: no near-threshold check, 1: check only, 2: check and record
#endif
constexpr int kTieHeaderWords = 4;  // count, blocks of k_dense_settle done, entries dropped (cumulative), 0

// Appends the (chain m, unit n_first + j) of every bit j of each lane's `near` to the tie list: one
// atomic per warp, then each lane's entries at its prefix offset.  Entries past the capacity are
// dropped (their float32 decisions stand) and counted by k_dense_settle.  All 32 lanes call it.
__device__ __forceinline__ void record_ties(uint32_t* ties, int64_t cap, uint32_t near, int64_t m,
                                            int64_t n_first) {
  const int lane = threadIdx.x & 31;
  const uint32_t cnt = (uint32_t)__popc(near);
  uint32_t incl = cnt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  uint32_t base = 0u;
  if (lane == 31) base = atomicAdd(ties, incl);
  base = __shfl_sync(0xffffffffu, base, 31);
  uint32_t idx = base + incl - cnt;
  uint2* entries = reinterpret_cast<uint2*>(ties + kTieHeaderWords);
  while (near) {
    const int j = __ffs(near) - 1;
    near &= near - 1u;
    if ((int64_t)idx < cap) entries[idx] = make_uint2((uint32_t)m, (uint32_t)(n_first + j));
    ++idx;
  }
}

// Tile t of a persistent CTA -> (m block, n block): the row blocks are taken
// `group` at a time and each group is walked row-fastest, so the tiles in
// flight at one time share one or two B column panels while the group's A
// row panels stay in L2 for the sweep over the group's columns.  The
// single-CTA kernel takes 16 row blocks of 128 rows; the CTA-pair kernel
// sizes its groups of 256-row blocks to about 32 MiB of A panels
// (group x 256 x K x 2 bytes), which measured lowest in DRAM bytes for both
// GEMMs of the 4096 x 8192 RBM (K = 4096: 16 blocks, K = 8192: 8 blocks;
// 64 MiB groups or a plain row-major walk re-read more).
constexpr int kGroupM = 16;
__device__ __forceinline__ void tile_coords(int t, int m_blocks, int n_blocks, int group, int& mb, int& nb) {
  const int per_group = group * n_blocks;
  const int g = t / per_group, w = t - g * per_group;
  const int rows = min(group, m_blocks - g * group);
  mb = g * group + w % rows;
  nb = w / rows;
}

// The 32 biases of a chunk (n_first % 32 == 0, bias 16-byte aligned): eight 16-byte loads, the same
// addresses in every lane; zeros without a bias.
__device__ __forceinline__ void load_bias32(const float* bias, int64_t n_first, float (&b)[32]) {
  if (!bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j) b[j] = 0.0f;
    return;
  }
  const float4* bq = reinterpret_cast<const float4*>(bias + n_first);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 v = __ldg(bq + q);
    b[4 * q] = v.x;
    b[4 * q + 1] = v.y;
    b[4 * q + 2] = v.z;
    b[4 * q + 3] = v.w;
  }
}

// Spin epilogue of one 32-column chunk of row m: bit j of the result is set when unit n_first + j samples
// -1.  +1 with probability sigmoid(2 field): u * (1 + e^(-2 field)) < 1 with u = uniform_open of the
// unit's Philox word (u is built with ALU operations, bit for bit the same value), or 2 field > logit.
// `near` receives the decisions within kNearTie of their threshold.
template <bool VARIATES>
__device__ __forceinline__ uint32_t spin_chunk(const DenseArgs& a, const float (&acc)[32], int64_t m,
                                               int64_t n_first, uint32_t sweep, const PhiloxKeys& keys,
                                               int64_t vs, uint32_t& near) {
  const int64_t gchain = a.chain_offset + m;
  const int64_t r0 = a.row0 + n_first;
  uint32_t down = 0u;
  near = 0u;
  if (VARIATES) {
    float b[32];
    load_bias32(a.bias, n_first, b);
    const float* vrow = a.variates + (vs * a.N + n_first) * a.M + m;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float field = __fadd_rn(acc[j], b[j]);
      const float d = __fsub_rn(__fmul_rn(2.0f, field), __ldg(vrow + (int64_t)j * a.M));
      down |= (d > 0.0f ? 0u : 1u) << j;
      if (TTHRML_DENSE_SETTLE) near |= (fabsf(d) < kNearTie ? 1u : 0u) << j;
    }
  } else if ((r0 & 3) == 0) {  // the chunk starts a Philox counter: word j % 4 of counter r0 / 4 + j / 4
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const u32x4 r = philox4x32_10(u32x4{(uint32_t)gchain, (uint32_t)((r0 >> 2) + q), sweep, kSaltDenseSpin}, keys);
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
      const float4 bq = a.bias ? __ldg(reinterpret_cast<const float4*>(a.bias + n_first) + q) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float b[4] = {bq.x, bq.y, bq.z, bq.w};
#if TTHRML_DENSE_F32X2
      // two units per packed instruction: t = u * (1 + 2^(-2 log2(e) field)), decided against 1
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int j = 4 * q + i;
        const float2 field = __fadd2_rn(make_float2(acc[j], acc[j + 1]), make_float2(b[i], b[i + 1]));
        const float2 x = __fmul2_rn(field, make_float2(-2.8853900817779268f, -2.8853900817779268f));
        float e0, e1;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x.y));
        const float2 u = __fadd2_rn(make_float2(__uint_as_float(0x3F800000u | (w[i] >> 9)),
                                                __uint_as_float(0x3F800000u | (w[i + 1] >> 9))),
                                    make_float2(-0.99999994039535522461f, -0.99999994039535522461f));
        const float2 t = __fmul2_rn(u, __fadd2_rn(make_float2(e0, e1), make_float2(1.0f, 1.0f)));
        down |= ((t.x < 1.0f ? 0u : 1u) | (t.y < 1.0f ? 0u : 2u)) << j;
        if (TTHRML_DENSE_SETTLE) {
          const float2 d = __fadd2_rn(t, make_float2(-1.0f, -1.0f));
          near |= ((fabsf(d.x) < kNearTie ? 1u : 0u) | (fabsf(d.y) < kNearTie ? 2u : 0u)) << j;
        }
      }
#else
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * q + i;
        const float field = __fadd_rn(acc[j], b[i]);
        const float t = uniform_open_alu(w[i]) * (1.0f + __expf(-2.0f * field));
        down |= (t < 1.0f ? 0u : 1u) << j;
        if (TTHRML_DENSE_SETTLE) near |= (fabsf(t - 1.0f) < kNearTie ? 1u : 0u) << j;
      }
#endif
    }
  } else {
    float b[32];
    load_bias32(a.bias, n_first, b);
    u32x4 r{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int64_t row = r0 + j;
      if (j == 0 || (row & 3) == 0)
        r = philox4x32_10(u32x4{(uint32_t)gchain, (uint32_t)(row >> 2), sweep, kSaltDenseSpin}, keys);
      const float field = __fadd_rn(acc[j], b[j]);
      const float t = uniform_open_alu(word_of(r, (int)(row & 3))) * (1.0f + __expf(-2.0f * field));
      down |= (t < 1.0f ? 0u : 1u) << j;
      if (TTHRML_DENSE_SETTLE) near |= (fabsf(t - 1.0f) < kNearTie ? 1u : 0u) << j;
    }
  }
  return down;
}

// Box-Muller on words 2p, 2p+1 of a counter: the normals of rows 4j+2p (cosine) and 4j+2p+1 (sine).
__device__ __forceinline__ void box_muller_pair(uint32_t w0, uint32_t w1, float& xc, float& xs) {
  const float rad = sqrtf(-2.0f * logf(uniform_open(w0)));
  float sn, cs;
#if TTHRML_DENSE_FAST_TRIG
  // theta = 2 pi u1 = phi + pi with phi = 2 pi (u1 - 1/2) in (-pi, pi), where the hardware sine and cosine
  // are accurate to ~5e-7 absolute: cos theta = -cos phi, sin theta = -sin phi
  __sincosf(6.2831853071795865f * (uniform_open_alu(w1) - 0.5f), &sn, &cs);
  xc = -rad * cs;
  xs = -rad * sn;
#else
  sincospif(2.0f * uniform_open(w1), &sn, &cs);
  xc = rad * cs;
  xs = rad * sn;
#endif
}

// Gaussian epilogue of one 32-column chunk: field * var + sqrt(var) * xi, xi the unit's normal from the
// counter (chain, row / 4, sweep, "DGAU") (or the uploaded normal).
template <bool VARIATES>
__device__ __forceinline__ void gauss_chunk(const DenseArgs& a, const float (&acc)[32], int64_t m,
                                            int64_t n_first, uint32_t sweep, const PhiloxKeys& keys, float inv,
                                            float sd_g, int64_t vs, float (&outf)[32]) {
  float b[32];
  load_bias32(a.bias, n_first, b);
  const int64_t gchain = a.chain_offset + m;
  const int64_t r0 = a.row0 + n_first;
  float xi[32];
  if (VARIATES) {
    const float* vrow = a.variates + (vs * a.N + n_first) * a.M + m;
#pragma unroll
    for (int j = 0; j < 32; ++j) xi[j] = __ldg(vrow + (int64_t)j * a.M);
  } else if ((r0 & 3) == 0) {  // the chunk starts a counter: rows 4q..4q+3 of the chunk share counter q
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const u32x4 r = philox4x32_10(u32x4{(uint32_t)gchain, (uint32_t)((r0 >> 2) + q), sweep, kSaltDenseGauss}, keys);
      box_muller_pair(r.x, r.y, xi[4 * q], xi[4 * q + 1]);
      box_muller_pair(r.z, r.w, xi[4 * q + 2], xi[4 * q + 3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int64_t row = r0 + j;
      const u32x4 r = philox4x32_10(u32x4{(uint32_t)gchain, (uint32_t)(row >> 2), sweep, kSaltDenseGauss}, keys);
      const int w = (int)((row >> 1) & 1) * 2;
      float xc, xs;
      box_muller_pair(word_of(r, w), word_of(r, w + 1), xc, xs);
      xi[j] = (row & 1) ? xs : xc;
    }
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float field = a.bias ? __fadd_rn(acc[j], b[j]) : acc[j];
    outf[j] = __fadd_rn(__fmul_rn(field, inv), __fmul_rn(sd_g, xi[j]));
  }
}

// Epilogue of one 32-column chunk of one row (chain m): draw and store.  The new value goes to the
// float32 copy (if any) and as `pieces` bf16 pieces: piece p = bf16(v - pieces 0..p-1), each remainder
// exact in float32, so three pieces carry all 24 significand bits.  A spin's +-1 is one bf16 piece
// (0x3F80 / 0xBF80) and zero remainders.
template <int FAMILY, bool VARIATES>
__device__ __forceinline__ void draw_chunk(const DenseArgs& a, const float (&acc)[32], int64_t m, int64_t n_first,
                                           uint32_t sweep, const PhiloxKeys& keys, float inv, float sd_g,
                                           int64_t vs) {
  __nv_bfloat16* row = a.out + m * (a.N * a.pieces) + n_first;
  if (FAMILY == TTHRML_SPIN) {
    uint32_t near;
    const uint32_t down = spin_chunk<VARIATES>(a, acc, m, n_first, sweep, keys, vs, near);
    if (TTHRML_DENSE_SETTLE == 2 && a.ties != nullptr &&
        __any_sync(0xffffffffu, near != 0u))  // rare: k_dense_settle decides these again from the exact field
      record_ties(a.ties, a.ties_cap, near, m, n_first);
    if (a.out_f32) {
      float4* df = reinterpret_cast<float4*>(a.out_f32 + m * a.N + n_first);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(0x3F800000u | (((down >> (4 * q + i)) & 1u) << 31));
        df[q] = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    uint32_t w[16];  // bf16 pairs (unit 2k in the low half)
#pragma unroll
    for (int k = 0; k < 16; ++k)
      w[k] = 0x3F803F80u | (((down >> (2 * k)) & 1u) << 15) | (((down >> (2 * k + 1)) & 1u) << 31);
    uint4* dst = reinterpret_cast<uint4*>(row);
#pragma unroll
    for (int q = 0; q < 4; ++q) dst[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    for (int p = 1; p < a.pieces; ++p) {
      uint4* z = reinterpret_cast<uint4*>(row + p * a.N);
#pragma unroll
      for (int q = 0; q < 4; ++q) z[q] = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  float outf[32];
  gauss_chunk<VARIATES>(a, acc, m, n_first, sweep, keys, inv, sd_g, vs, outf);
  if (a.out_f32) {
    float4* df = reinterpret_cast<float4*>(a.out_f32 + m * a.N + n_first);
#pragma unroll
    for (int q = 0; q < 8; ++q) df[q] = make_float4(outf[4 * q], outf[4 * q + 1], outf[4 * q + 2], outf[4 * q + 3]);
  }
  for (int p = 0; p < a.pieces; ++p) {
    __align__(16) __nv_bfloat16 outv[32];
    const bool last = p + 1 == a.pieces;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      outv[j] = __float2bfloat16_rn(outf[j]);
      if (!last) outf[j] = __fsub_rn(outf[j], __bfloat162float(outv[j]));
    }
    uint4* dst = reinterpret_cast<uint4*>(row + p * a.N);
    const uint4* srcv = reinterpret_cast<const uint4*>(outv);
#pragma unroll
    for (int q = 0; q < 4; ++q) dst[q] = srcv[q];
  }
}

}  // namespace
}  // namespace tthrml
