// Building blocks of the tensor-core kernels (tcgen05): bounded mbarrier waits, TMA tile loads, shared-memory
// descriptors, TMEM loads, CTA-pair and cluster helpers, and the driver entry point that encodes tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>

#include "common.cuh"

namespace tthrml {
namespace {

constexpr long long kWaitCycles = 4ll << 30;  // about two seconds at 2 GHz

enum : int { kErrNone = 0, kErrFullWait = 1, kErrEmptyWait = 2, kErrAccWait = 3 };

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the phase of `parity` to complete; false when the clock limit expires.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_test(bar, parity)) {
    if (clock64() - t0 > kWaitCycles) return false;
  }
  return true;
}

// The same for a whole warp, all lanes polling: the shortest way to the answer.
__device__ __forceinline__ bool mbar_wait_all(uint64_t* bar, uint32_t parity) {
  const bool ok = mbar_wait(bar, parity);
  return __all_sync(0xffffffffu, (int)ok) != 0;
}
// The same, one lane polling, for warps that wait long: 32 polling lanes of each slow down the barriers that the loads and
// MMAs go by (8-bit tiles of 128 x 64: 318 clocks per 128 columns instead of 430).
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity);
  return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
}
// True in one lane of a whole warp.  A warp that loads or multiplies walks its loop together and this lane issues: addresses
// and descriptors then stay in uniform registers, where a loop of one thread moves each of them over for every instruction
// (8-bit tiles of 128 x 64: 53 clocks per MMA and 370 beside them; 128 x 64 x 8192 columns 23.7 us, now 15.5).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

// UMMA shared-memory descriptor of a K-major tile in the 128B-swizzle layout
// written by TMA (rows of 128 B, 8-row groups 1024 B apart): start address,
// leading offset 16 B, stride offset 1024 B, descriptor version 1, layout 2.
__device__ __forceinline__ uint64_t umma_desc_sw128(const void* tile) {
  const uint64_t addr = (uint64_t)(smem_u32(tile) >> 4) & 0x3FFFull;
  return addr | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// The same without the wait: v holds its values only after tmem_wait.
__device__ __forceinline__ void tmem_load32_async(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
// Waits for the warp's loads; every use of v stays behind it.
template <int N>
__device__ __forceinline__ void tmem_wait(float (&v)[N][32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int q = 0; q < N; ++q)
    asm volatile(""
                 : "+f"(v[q][0]), "+f"(v[q][1]), "+f"(v[q][2]), "+f"(v[q][3]), "+f"(v[q][4]), "+f"(v[q][5]), "+f"(v[q][6]),
                   "+f"(v[q][7]), "+f"(v[q][8]), "+f"(v[q][9]), "+f"(v[q][10]), "+f"(v[q][11]), "+f"(v[q][12]),
                   "+f"(v[q][13]), "+f"(v[q][14]), "+f"(v[q][15]), "+f"(v[q][16]), "+f"(v[q][17]), "+f"(v[q][18]),
                   "+f"(v[q][19]), "+f"(v[q][20]), "+f"(v[q][21]), "+f"(v[q][22]), "+f"(v[q][23]), "+f"(v[q][24]),
                   "+f"(v[q][25]), "+f"(v[q][26]), "+f"(v[q][27]), "+f"(v[q][28]), "+f"(v[q][29]), "+f"(v[q][30]),
                   "+f"(v[q][31]));
}

// 16 columns, for epilogues that hold many values already.
__device__ __forceinline__ void tmem_load16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// Two float32 operations in one instruction, each rounded by itself.
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float& a0, float& a1, float b) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b));
}
// a b + c
__device__ __forceinline__ void fma2(float a0, float a1, float b, float c, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b), "f"(c));
}

constexpr uint32_t kPeerMask = 0xFEFFFFFFu;  // clears the CTA-rank bit of a shared::cluster address

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_id_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t n_clusters_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();  // the barrier is a whole warp's
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_leader, int c0,
                                                 int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar_leader), "r"(c0), "r"(c1)
      : "memory");
}
// arrives (once all earlier MMAs of this thread are done) on the barrier at this offset in both CTAs
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)0x3)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & kPeerMask) : "memory");
}

// Shared-memory descriptor of an MN-major tile in the 128-byte swizzle: boxes of 64 units x 64 chains (8 KiB), so
// groups of 64 units are 8192 bytes apart (leading offset) and groups of 8 chains 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t umma_desc_mn128(const void* tile) {
  const uint64_t addr = (uint64_t)(smem_u32(tile) >> 4) & 0x3FFFull;
  return addr | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}
__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u),
      "r"(0u), "r"(0u));
}

constexpr int kTurnPitch = 80;  // bytes per row of a warp's staged 32 x 64 bytes: rows 20 banks apart
// Stores 32 staged rows of `bytes` each (a power of two up to 64) from column byte `at` of the output rows m0 .. m0 + 31, V at
// a time: a warp's store covers whole pieces of a few rows, where a store of every lane's own row would touch 32 lines.
template <typename V>
__device__ __forceinline__ void drain(const unsigned char* turn, int bytes, unsigned char* out, int64_t pitch, int64_t at,
                                      int m0, int M, int live_bytes) {
  const int lane = threadIdx.x & 31, per_row = bytes / (int)sizeof(V), rows = 32 / per_row;
  const int k = (lane % per_row) * (int)sizeof(V);
  if (k >= live_bytes) return;
#pragma unroll 4
  for (int r = lane / per_row; r < 32 && m0 + r < M; r += rows)
    *reinterpret_cast<V*>(out + (int64_t)(m0 + r) * pitch + at + k) = *reinterpret_cast<const V*>(turn + r * kTurnPitch + k);
}
// words: this lane's row, N16 pieces of 16 bytes.  Every lane calls it; the rows are m0 .. m0 + 31, `align` their alignment.
template <int N16>
__device__ __forceinline__ void store_rows(const uint4 (&words)[N16], unsigned char* turn, unsigned char* out, int64_t pitch,
                                           int64_t at, int m0, int M, int live_bytes, int align) {
  const int lane = threadIdx.x & 31;
  uint4* mine = reinterpret_cast<uint4*>(turn + lane * kTurnPitch);
#pragma unroll
  for (int q = 0; q < N16; ++q) mine[q] = words[q];
  __syncwarp();
  if (live_bytes < 16 * N16) align = align < 4 ? align : (live_bytes % 4 == 0 ? 4 : 2);
  if (align >= 16)
    drain<uint4>(turn, 16 * N16, out, pitch, at, m0, M, live_bytes);
  else if (align >= 8)
    drain<uint2>(turn, 16 * N16, out, pitch, at, m0, M, live_bytes);
  else if (align >= 4)
    drain<uint32_t>(turn, 16 * N16, out, pitch, at, m0, M, live_bytes);
  else
    drain<uint16_t>(turn, 16 * N16, out, pitch, at, m0, M, live_bytes);
  __syncwarp();
}

// store_rows of 64 whole bytes to rows that start on 16 bytes.
__device__ __forceinline__ void store_rows64(const uint4 (&words)[4], uint32_t turn, unsigned char* out, int64_t pitch, int m0,
                                             int M) {
  const uint32_t lane = threadIdx.x & 31, mine = turn + lane * kTurnPitch;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + 16 * q), "r"(words[q].x), "r"(words[q].y), "r"(words[q].z),
                 "r"(words[q].w)
                 : "memory");
  __syncwarp();
  const int r0 = (int)lane >> 2;
  unsigned char* o = out + (int64_t)(m0 + r0) * pitch + 16 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(turn + (r0 + 8 * i) * kTurnPitch + 16 * (lane & 3))
                 : "memory");
    if (m0 + r0 + 8 * i < M) *reinterpret_cast<uint4*>(o + (int64_t)(8 * i) * pitch) = v;
  }
  __syncwarp();
}

// 32 values of each of a warp's rows m0 + lane, from column n on, to 16-bit or float32 rows.
__device__ __forceinline__ void store_values(const float (&v)[32], int32_t dtype, unsigned char* turn, unsigned char* out,
                                             int64_t ld, int64_t n, int m0, int M, int live, int align) {
  if (dtype == TTHRML_DT_F32) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = make_uint4(__float_as_uint(v[16 * half + 4 * q]), __float_as_uint(v[16 * half + 4 * q + 1]),
                          __float_as_uint(v[16 * half + 4 * q + 2]), __float_as_uint(v[16 * half + 4 * q + 3]));
      const int left = min(16, live - 16 * half);
      if (left > 0) store_rows<4>(w, turn, out, ld * 4, 4 * (n + 16 * half), m0, M, 4 * left, align);
    }
    return;
  }
  uint4 w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = v[8 * q + 2 * j], hi = v[8 * q + 2 * j + 1];
      if (dtype == TTHRML_DT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    w[q] = make_uint4(p[0], p[1], p[2], p[3]);
  }
  store_rows<4>(w, turn, out, ld * 2, 2 * n, m0, M, 2 * live, align);
}

// Rows of 128 bytes on their way out through a bulk tensor store: a warp's 32 rows (a row per lane) in a buffer of 4096 bytes
// (1024-byte aligned), in the 128-byte swizzle, which both the lanes' writes and the store's reads spread over all banks.  The
// lane that issues the stores waits for their reads before a buffer is written again.
constexpr int kOutBytes = 32 * 128;
template <int N>
__device__ __forceinline__ void stage_row(uint32_t buffer, const uint4 (&w)[N], uint32_t first = 0) {  // N of its eight pieces
  const uint32_t lane = threadIdx.x & 31, row = buffer + lane * 128;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + 16 * ((first + j) ^ (lane & 7))), "r"(w[j].x), "r"(w[j].y), "r"(w[j].z),
                 "r"(w[j].w)
                 : "memory");
}
// To rows `row` .. row + 31 of plane `plane` from column `column` on; add: onto the float32 values there.
__device__ __forceinline__ void send_rows(const CUtensorMap* map, uint32_t buffer, int column, int row, int plane = 0,
                                          bool add = false) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (add)
      asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                   "r"(buffer), "r"(column), "r"(row), "r"(plane)
                   : "memory");
    else
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(buffer),
                   "r"(column), "r"(row), "r"(plane)
                   : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// All but the last `PENDING` stores of this warp have read their buffers.
template <int PENDING>
__device__ __forceinline__ void sent_rows_read() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory");
  __syncwarp();
}
__device__ __forceinline__ void sent_rows_done() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
}
// N 16-byte words of 8 N values rounded to 16 bits.
template <int N>
__device__ __forceinline__ void pack_row(const float* v, int32_t dtype, uint4* w) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (dtype == TTHRML_DT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * q + 2 * j], v[8 * q + 2 * j + 1]);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[8 * q + 2 * j], v[8 * q + 2 * j + 1]);
        p[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    w[q] = make_uint4(p[0], p[1], p[2], p[3]);
  }
}

// --- host side --------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_fn(EncodeTiledFn* out) {
  static EncodeTiledFn fn = nullptr;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) {
      set_error("cuTensorMapEncodeTiled is unavailable (%s)", cudaGetErrorString(e));
      return TTHRML_ERR_CUDA;
    }
    fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  *out = fn;
  return TTHRML_OK;
}

// Tensor map of output matrices [planes][rows][cols], rows `ld` and planes `plane` elements apart, for stores of 32 rows x
// 128 bytes; false where the rows do not start on 16 bytes (or are too far apart).
inline bool make_out_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int32_t dtype,
                         int64_t planes = 1, int64_t plane = 0) {
  const int64_t bytes = dtype == TTHRML_DT_F32 ? 4 : 2, apart = planes > 1 ? plane : rows * ld;
  EncodeTiledFn fn;
  if ((uintptr_t)base % 16 || ld * bytes % 16 || apart * bytes % 16 || ld * bytes >= (int64_t)1 << 40 ||
      apart * bytes >= (int64_t)1 << 40 || encode_fn(&fn))
    return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * bytes), (cuuint64_t)(apart * bytes)};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / bytes), 32u, 1u};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type = dtype == TTHRML_DT_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == TTHRML_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clocks of a block of the main loop (128 bytes of K) that brings `bytes` into each of `ctas` SMs at once: an SM takes in 68
// bytes a clock, all of them 7900 from L2; mma: the multiplications' own, or what it takes to issue them.
inline int64_t block_clocks(int64_t bytes, int64_t ctas, int64_t mma) {
  return std::max({mma, bytes / 68, bytes * ctas / 7900});
}

// What a launch of fn in clusters needs to know about the current device, asked once per device and function:
// the raised shared-memory limit and how many clusters are resident at once.
struct ClusterFit {
  int sms, clusters;
};
inline int cluster_fit(const void* fn, unsigned cluster, unsigned threads, int smem, ClusterFit* out) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*, unsigned, int>, ClusterFit> known;
  static std::map<std::pair<int, const void*>, int> limits;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(dev, fn, cluster, smem);
  const auto it = known.find(key);
  if (it != known.end()) {
    *out = it->second;
    return TTHRML_OK;
  }
  ClusterFit f = {0, 0};
  int& limit = limits[std::make_pair(dev, fn)];  // never lowered: earlier launches may have needed more
  e = cudaDeviceGetAttribute(&f.sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && smem > limit) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) limit = smem;
  }
  if (e != cudaSuccess) return cuda_status(e, "kernel attributes");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(cluster, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(&f.clusters, fn, &cfg);
  if (e != cudaSuccess) return cuda_status(e, "cudaOccupancyMaxActiveClusters");
  if (f.clusters < 1) {
    set_error("no cluster of %u blocks fits on this device", cluster);
    return TTHRML_ERR_UNSUPPORTED;
  }
  known.emplace(key, f);
  *out = f;
  return TTHRML_OK;
}

// Launches fn on a one-dimensional grid of clusters.  early: the kernel may start while the one before it on the stream
// still runs (programmatic dependent launch); it waits for it by wait_for_previous_kernel() before it reads what that
// kernel writes.
inline int launch_clusters(const void* fn, unsigned grid, unsigned cluster, unsigned threads, int smem, void** params,
                           cudaStream_t st, const char* what, bool early = false) {
  ClusterFit fit;
  const int rc = cluster_fit(fn, cluster, threads, smem, &fit);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, params);
  if (e != cudaSuccess) return cuda_status(e, what);
  return launch_status(what);
}

}  // namespace
}  // namespace tthrml
