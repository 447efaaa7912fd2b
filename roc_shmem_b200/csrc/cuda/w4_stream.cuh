// w4_stream.cuh — out[T, N] = x[T, K] · w[N, K]^T with weights of 4 bits on the tcgen05 tensor cores:
//
//   w[n, k] = (q[n, k] - z[n, k / group]) * s[n, k / group],   q in 0..15, z in 0..15 (8 where there is none), s bf16
//
// The weights are read once, half a byte each, and what counts besides is how many instructions turn one into an operand.  A
// tile is 128 weight rows (the MMA's M) times up to 64 tokens (its N); a k-block is 128 columns.  A thread widens a row of a
// k-block: a nibble becomes a bf16 by or-ing it into the mantissa of 128, and 128 + q - (128 + z) is exact.  The pairs that come
// out, columns (0,4) (1,5) (2,6) (3,7) of every eight, go to tensor memory as operand A as they are, and the activations'
// columns are put into the same order where they lie in shared memory.  The scales never touch the weights: each group has an
// accumulator of its own, which the thread of the row multiplies by its scale and adds up in fp32 registers.
//
//   warp 0      TMA producer: {128 rows x 128 bytes of weights, tokens x 256 columns} per stage, i.e. two k-blocks (with rows of 64
//               bytes the TMA unit's requests, one per row, were the limit); plain loads of local memory
//   warp 1      MMA issuer: tcgen05.mma M128 x N=tokens x K16, A in tensor memory, B in shared memory
//   then        two to five groups of four warps: each widens every second to fifth k-block and orders its activations
//   last 4      add the accumulators up
//
// From a k-block's arrival to its sums it takes a warp of each kind some 900 cycles, and HBM brings an SM the 8 KiB of the next in 370: so several
// are on their way (kDepth stages in tensor memory, of two each; one stage where its accumulators take most: 64 tokens in groups of 64,
// 32 in groups of 32), in the hands of different warps.  The ALU is behind that: seven shifts and
// logical operations for eight weights at half the rate of the other pipes, 230 cycles for a k-block.
//
// A cluster of up to 8 CTAs splits the columns of a tile where tiles are few, and adds the parts through distributed shared memory
// in the CTAs' order: reproducible bits, no workspace.  Every wait is bounded (see gemm_core.cuh).
#pragma once
#include <cuda_bf16.h>

#include <cstring>

#include "gemm_pair.cuh"
#include "tma_host.h"

namespace bshmem {
namespace w4 {

using gemm::Guard;
using gemm2::cluster_ctarank;
using gemm2::cluster_sync_all;
using gemm2::ld_cluster_f4;
using gemm2::mapa;
using gemm2::warp_wait;

constexpr int ROWS = 128, BK = 128;                  // weight rows of a tile, columns of a k-block
constexpr int MAX_STAGES = 9, MAX_DEPTH = 3;
constexpr int WIDENERS = 4, ADDERS = 4;              // warps of a group that widens, and warps that add up
constexpr uint32_t W_BYTES = ROWS * BK;              // 16 KiB of weights per stage: two k-blocks
constexpr uint32_t CTRL_BYTES = 512;
constexpr uint32_t SMEM_BYTES = 224u << 10;          // one CTA has an SM, all of its tensor memory too
constexpr uint32_t TMEM_COLS = 512;
enum ErrSite : int { ERR_PRODUCER_EMPTY = 401, ERR_MMA_A = 402, ERR_WIDEN_FULL = 403, ERR_WIDEN_ADDED = 404, ERR_ADD_DONE = 405 };

struct Params {
  CUtensorMap map_w, map_x;      // weights [N, K / 2] bytes, box {128, 128}; tokens [T, K], box {64, nt}
  const void* x; long long ldx;  // for the host
  const __nv_bfloat16* s;
  const uint8_t* z;              // null: 8 everywhere
  __nv_bfloat16* out;            // [T, N]
  long long ldo;
  int T, N, K, group;
  int split;
  unsigned long long timeout_ns;
};

__device__ int error_word;        // site of the first wait that ran out, 0: none

__host__ __device__ constexpr uint32_t stage_bytes(int nt) { return W_BYTES + (uint32_t)nt * BK * 4; }
__host__ __device__ constexpr int stages(int nt) {
  return (SMEM_BYTES - CTRL_BYTES - 1024) / stage_bytes(nt) < MAX_STAGES ? (SMEM_BYTES - CTRL_BYTES - 1024) / stage_bytes(nt) : MAX_STAGES;
}
// Stages in tensor memory, each with two A buffers of 64 columns and `subs` accumulators of nt for either.
__host__ __device__ constexpr int block_cols(int nt, int subs) { return 2 * (64 + subs * nt); }
__host__ __device__ constexpr int depth(int nt, int subs) {
  return TMEM_COLS / block_cols(nt, subs) < MAX_DEPTH ? TMEM_COLS / block_cols(nt, subs) : MAX_DEPTH;
}
// Groups that widen: no more than there are k-blocks in tensor memory, or a group could ask about a buffer's round before last and take
// the answer for its last one; three for 64 tokens, whose sums take more registers; five for 16 tokens in groups of 128 columns and
// more, whose sums take fewest (7168 rows of 8192, one token: 14.1 us with four, 13.7 with five or six; 4096 of 4096: 6.8, 6.8, 7.2).
__host__ __device__ constexpr int widen_groups(int nt, int subs) {
  const int most = nt == 64 ? 3 : nt == 16 && subs == 1 ? 5 : 4;
  return 2 * depth(nt, subs) < most ? 2 * depth(nt, subs) : most;
}
__host__ __device__ constexpr int threads(int nt, int subs) { return 32 * (2 + WIDENERS * widen_groups(nt, subs) + ADDERS); }

__device__ __forceinline__ __nv_bfloat162 as_pair(uint32_t w) {
  __nv_bfloat162 p;
  memcpy(&p, &w, 4);
  return p;
}
__device__ __forceinline__ uint32_t as_word(__nv_bfloat162 p) {
  uint32_t w;
  memcpy(&w, &p, 4);
  return w;
}
// Eight nibbles n0 .. n7 as bf16 pairs (n0, n4), (n1, n5), (n2, n6), (n3, n7), less `off` = 128 + z in both halves.
__device__ __forceinline__ void widen(uint32_t w, __nv_bfloat162 off, uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(w >> (4 * i)));      // (w & mask) | 128.0 in one
    o[i] = as_word(__hsub2(as_pair(v), off));
  }
}
// The same order of eight activations.
__device__ __forceinline__ uint4 pair_up(uint4 v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

struct Smem {
  uint32_t base, stage, ctrl;    // 1024-byte aligned base, bytes of a stage, control block
  uint8_t* gen;                  // generic pointer to the control block
  __device__ __forceinline__ uint32_t w(int s) const { return base + s * stage; }
  __device__ __forceinline__ uint32_t x(int s) const { return base + s * stage + W_BYTES; }
  __device__ __forceinline__ uint32_t full(int s) const { return ctrl + 8 * s; }
  __device__ __forceinline__ uint32_t empty(int s) const { return ctrl + 8 * (MAX_STAGES + s); }
  __device__ __forceinline__ uint32_t wide(int b) const { return ctrl + 8 * (2 * MAX_STAGES + b); }                  // A buffer b is written
  __device__ __forceinline__ uint32_t done(int b) const { return ctrl + 8 * (2 * MAX_STAGES + MAX_DEPTH + b); }      // its MMAs are done
  __device__ __forceinline__ uint32_t added(int b) const { return ctrl + 8 * (2 * MAX_STAGES + 2 * MAX_DEPTH + b); } // its sums are added up
  __device__ __forceinline__ uint32_t tmem_slot() const { return ctrl + 8 * (2 * MAX_STAGES + 3 * MAX_DEPTH); }
  __device__ __forceinline__ volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(gen + 8 * (2 * MAX_STAGES + 3 * MAX_DEPTH + 1)); }
};

// kNt: tokens of the tile (16, 32 or 64).  kSubs: groups of a k-block (1 for groups of 128 columns and more, 2, 4).
template <int kNt, int kSubs>
__global__ void __launch_bounds__(threads(kNt, kSubs), 1) w4_stream_kernel(const __grid_constant__ Params p) {
  constexpr int kDepth = depth(kNt, kSubs), kCols = block_cols(kNt, kSubs);        // columns of a stage: A, then its accumulators
  constexpr int kStages = stages(kNt), kGroups = widen_groups(kNt, kSubs);
  // A wait knows a barrier's rounds by their parity only, so nobody may come to one two rounds early.  A group is (kGroups + 1) / 2 stages
  // at most behind its last k-block, when it knew all sums of kDepth stages before that to be added up (and so their loads, too).
  constexpr int kStride = (kGroups + 1) / 2;
  static_assert(kDepth >= kStride && kStages >= kStride + kDepth, "rounds of the barriers");
  extern __shared__ uint8_t smem_raw[];
  Smem L;
  {
    const uint32_t r = ptx::smem_u32(smem_raw);
    L.base = (r + 1023u) & ~1023u;
    L.stage = stage_bytes(kNt);
    L.ctrl = L.base + kStages * L.stage;
    L.gen = smem_raw + (L.ctrl - r);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, split = p.split;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)(blockIdx.x / split) * ROWS, tok0 = (int)blockIdx.y * kNt;
  const int pairs = (p.K + 2 * BK - 1) / (2 * BK), kb0 = pairs * rank / split * 2, kb1 = pairs * (rank + 1) / split * 2;       // whole stages
  Guard g{&error_word, L.abort_flag(), p.timeout_ns};

  if (threadIdx.x == 0) {
    *L.abort_flag() = 0;
    for (int s = 0; s < kStages; ++s) { ptx::mbar_init(L.full(s), 1); ptx::mbar_init(L.empty(s), 1); }
    for (int b = 0; b < kDepth; ++b) { ptx::mbar_init(L.wide(b), 2 * WIDENERS); ptx::mbar_init(L.done(b), 1); ptx::mbar_init(L.added(b), ADDERS); }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&p.map_w);
    ptx::prefetch_tensormap(&p.map_x);
  }
  if (warp == 1) {
    ptx::tmem_alloc(L.tmem_slot(), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  // The first weights start on their way to L2 while the previous kernel still runs; a prefetch reads nothing.
  if (warp == 2 && lane == 0)
    for (int kb = kb0; kb < min(kb1, kb0 + 2 * kStages); kb += 2) ptx::tma_prefetch_2d(&p.map_w, kb * (BK / 2), n0);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // All of tensor memory begins at column 0.  As a constant it keeps the addresses of the MMAs in uniform registers: as a value from
  // memory they were moved there one by one, some 60 cycles for each MMA.
  constexpr uint32_t tmem = 0;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  if (warp == 0) {
    const bool leader = ptx::elect_one();
    int s = 0; uint32_t ph = 0;
    for (int kb = kb0; kb < kb1; kb += 2) {
      if (!warp_wait(L.empty(s), ph ^ 1, g, ERR_PRODUCER_EMPTY)) break;
      if (leader) {
        ptx::mbar_arrive_expect_tx(L.full(s), L.stage);
        ptx::tma_load_2d(L.w(s), &p.map_w, L.full(s), kb * (BK / 2), n0);
#pragma unroll
        for (int a = 0; a < 4; ++a) ptx::tma_load_2d(L.x(s) + a * kNt * 128, &p.map_x, L.full(s), kb * BK + a * 64, tok0);
      }
      if (++s == kStages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    const bool leader = ptx::elect_one();
    constexpr uint32_t idesc = ptx::umma_idesc(1, 1, ROWS, kNt);
    // Two k-blocks at once: a wait that is over still takes 150 cycles, a commit 50.
    int s = 0, b = 0; uint32_t ph = 0;                // buffer b in its round ph
    for (int kb = kb0; kb < kb1; kb += 2) {
      if (!warp_wait(L.wide(b), ph, g, ERR_MMA_A)) break;
      ptx::tc_fence_after();
      if (leader) {
        const uint32_t a = tmem + b * kCols, d = a + 128;
        const uint64_t dx = ptx::umma_desc_sw128(L.x(s));
#pragma unroll
        for (int k = 0; k < 2 * BK / 16; ++k) {
          constexpr int kPer = BK / 16 / kSubs;       // MMAs of a group
          umma_f16_ts(d + k / kPer * kNt, a + k * 8, dx + (k / 4) * (kNt * 128 / 16) + (k % 4) * 2, idesc, k % kPer ? 1u : 0u);
        }
        ptx::umma_commit(L.done(b));
        ptx::umma_commit(L.empty(s));
      }
      __syncwarp();
      if (++s == kStages) s = 0;
      if (++b == kDepth) { b = 0; ph ^= 1; }
    }
  } else if (warp < 2 + WIDENERS * kGroups) {
    // a thread widens its row of every kGroups-th k-block
    const int quarter = warp & 3, group = (warp - 2) / 4, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int groups = p.K / p.group, mine = (threadIdx.x - 64) % 128 * 16, tokens = min(kNt, p.T - tok0);
    const uint8_t* const z = p.z ? p.z + (long long)min(n0 + row, p.N - 1) * groups : nullptr;
    uint32_t zp[kSubs];                               // of the k-block's groups
    auto load = [&](int kb) {
#pragma unroll
      for (int j = 0; j < kSubs; ++j) zp[j] = z ? z[min(kSubs == 1 ? kb * BK / p.group : kb * kSubs + j, groups - 1)] : 8;
    };
    load(kb0 + group);
    int s = group / 2; uint32_t ph = 0;
    for (int i = group; i < kb1 - kb0; i += kGroups) {
      const int kb = kb0 + i, b = i / 2 % kDepth;
      if (!warp_wait(L.full(s), ph, g, ERR_WIDEN_FULL)) break;
      __nv_bfloat162 off[kSubs];
#pragma unroll
      for (int j = 0; j < kSubs; ++j) off[j] = as_pair(0x43004300u | zp[j] | zp[j] << 16);
      if (z) load(min(kb + kGroups, kb1 - 1));
      const uint32_t from = L.w(s) + row * 128, x = L.x(s) + (kb & 1) * kNt * 256 + mine;
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = ld_shared_v4(from + ((((kb & 1) * 4 + j) ^ (row & 7)) << 4));      // the stage's 128-byte swizzle
#pragma unroll
      for (int e = 0; e < kNt * BK * 2; e += 128 * 16) {
        if ((e + mine) / 128 % kNt < tokens) st_shared_v4(x + e, pair_up(ld_shared_v4(x + e)));          // the others are zero
      }
      ptx::fence_proxy_async_smem();                  // the MMAs read the activations through the async proxy
      const uint32_t to = tmem + lanes + b * kCols + (kb & 1) * 64;
      bool free = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t o[32];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const __nv_bfloat162 f = off[(h * 2 + j) * kSubs / 4];
          widen(w[h * 2 + j].x, f, o + j * 16);
          widen(w[h * 2 + j].y, f, o + j * 16 + 4);
          widen(w[h * 2 + j].z, f, o + j * 16 + 8);
          widen(w[h * 2 + j].w, f, o + j * 16 + 12);
        }
        if (h == 0) {                                 // the buffer's last k-block is multiplied and its sums are read
          free = warp_wait(L.added(b), (i / 2 / kDepth & 1) ^ 1, g, ERR_WIDEN_ADDED);
          ptx::tc_fence_after();
        }
        if (free) tmem_st_32x32b_x32(to + h * 32, o);
      }
      if (!free) break;
      tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(L.wide(b));
      // kGroups k-blocks on: as many halves of stages
      s = (i + kGroups) / 2 % kStages;
      ph = (i + kGroups) / 2 / kStages & 1;
    }
  } else {
    // a thread adds up its row's accumulators
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int groups = p.K / p.group, tokens = min(kNt, p.T - tok0);
    const unsigned short* const scales = reinterpret_cast<const unsigned short*>(p.s) + (long long)min(n0 + row, p.N - 1) * groups;
    float2 acc[kNt / 2];
#pragma unroll
    for (int j = 0; j < kNt / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    // The scales of eight groups ahead: a load takes as long as a k-block or two.
    constexpr int kBatch = 8 / kSubs;                 // k-blocks
    unsigned short sc[8], next[8];                    // as they come: a conversion would wait for its load
    auto load = [&](int kb) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        next[j] = scales[min(kSubs == 1 ? (kb + j) * BK / p.group : kb * kSubs + j, groups - 1)];
    };
    load(kb0);
    bool ok = true;
    int b = 0; uint32_t ph = 0;
    for (int first = kb0; ok && first < kb1; first += kBatch) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = next[j];
      load(first + kBatch);
#pragma unroll
      for (int u = 0; u < kBatch; u += 2) {
        if (!ok || first + u >= kb1) break;
        ok = warp_wait(L.done(b), ph, g, ERR_ADD_DONE);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + lanes + b * kCols + 128;
#pragma unroll
        for (int j = 0; j < 2 * kSubs; ++j)
#pragma unroll
          for (int c = 0; c < kNt; c += 16) {
            uint32_t v[16];
            ptx::tmem_ld_32x32b_x16(d + j * kNt + c, v);
            ptx::tmem_ld_wait();
            const float scale = __uint_as_float((uint32_t)sc[u * kSubs + j] << 16);
            const float2 f = make_float2(scale, scale);
#pragma unroll
            for (int t = 0; t < 8; ++t)
              acc[c / 2 + t] = fma2(f, make_float2(__uint_as_float(v[2 * t]), __uint_as_float(v[2 * t + 1])), acc[c / 2 + t]);
          }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(L.added(b));
        if (++b == kDepth) { b = 0; ph ^= 1; }
      }
    }
    if (ok) {
      if (split == 1) {
        __nv_bfloat16* out = p.out + n0 + row;
#pragma unroll
        for (int t = 0; t < kNt; ++t)                 // 32 lanes = 64 neighbouring bytes of a token's row
          if (n0 + row < p.N && t < tokens) out[(tok0 + t) * p.ldo] = __float2bfloat16_rn(t & 1 ? acc[t / 2].y : acc[t / 2].x);
      } else {
        // the part as [token][row] floats over the stages: all their loads have landed and all MMAs have read them
#pragma unroll
        for (int t = 0; t < kNt; ++t)
          if (t < tokens)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(L.base + (t * ROWS + row) * 4), "f"(t & 1 ? acc[t / 2].y : acc[t / 2].x) : "memory");
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (split > 1) {
    cluster_sync_all();
    if (!*L.abort_flag()) {
      // four rows of a token per thread; the tokens go round the cluster's CTAs
      const int tokens = min(kNt, p.T - tok0);
      for (int t = rank + warp * split; t < tokens; t += split * (threads(kNt, kSubs) / 32)) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < split; ++r) {
          const float4 a = ld_cluster_f4(mapa(L.base + t * (ROWS * 4) + lane * 16, r));
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
        }
        const float f[4] = {v.x, v.y, v.z, v.w};
        __nv_bfloat16* dst = p.out + (tok0 + t) * p.ldo + n0 + lane * 4;
        if (p.N % 4 == 0) {                           // the rows of `out` begin on 8 bytes
          if (n0 + lane * 4 < p.N)
            *reinterpret_cast<uint2*>(dst) = make_uint2(gemm::pack_bf16(f[0], f[1]), gemm::pack_bf16(f[2], f[3]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n0 + lane * 4 + j < p.N) dst[j] = __float2bfloat16_rn(f[j]);
        }
      }
    }
    cluster_sync_all();                               // nobody's shared memory goes away while it is being read
  }
  if (*L.abort_flag()) {
    // let copies and MMAs that are still in flight land before shared and tensor memory go away
    const unsigned long long t0 = ptx::globaltimer();
    while (ptx::globaltimer() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace w4
}  // namespace bshmem
