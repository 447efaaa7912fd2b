// gemm_w4.cu — out[T, N] = x[T, K] · w[N, K]^T for few tokens with weights of 4 bits:
//
//   w[n, k] = (q[n, k] - z[n, k / group]) * s[n, k / group],   q in 0..15, z in 0..15 (8 where there is none), s bf16
//
// q: [N, K/2] bytes, the low half of a byte is the column of even number; s, z: [N, K/group].
//
// Few tokens are bound by the weights, half a byte each, so what counts is that they stream and that turning them into operands
// takes few instructions.  A warp has 16 weight rows (mma.sync m16n8k16, the rows are M, up to 8 tokens are N) and reads 64
// contiguous bytes of each per step of 128 columns, 16 per lane.  The order of the columns inside a product is free as long as
// both operands have the same, so each lane multiplies the columns that it happens to hold.  A nibble becomes a bf16 by or-ing it
// into the mantissa of 128; 128 + q - (128 + z) is exact.  The group's scale multiplies the group's fp32 partial sum: the weight
// itself is never rounded.  Eight warps split the columns, and clusters of blocks too where rows are few.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tma_host.h"

using namespace bshmem;

namespace {

constexpr int kWarps = 8;
constexpr int kStep = 128;                            // columns of a step

struct FewParams {
  const __nv_bfloat16* x;
  const uint8_t* q;
  const __nv_bfloat16* s;
  const uint8_t* z;                                   // null: 8 everywhere
  __nv_bfloat16* out;
  long long ldx, ldo;
  int T, N, K, group;
  int split;                                          // blocks of a cluster that share a tile's columns
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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
__device__ __forceinline__ void widen(uint32_t w, __nv_bfloat162 off, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 d = __hsub2(as_pair(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u), off);
    o[i] = as_word(d);
  }
}
// The same order of eight activations.
__device__ __forceinline__ void pair_up(uint4 v, uint32_t (&o)[4]) {
  o[0] = __byte_perm(v.x, v.z, 0x5410);
  o[1] = __byte_perm(v.x, v.z, 0x7632);
  o[2] = __byte_perm(v.y, v.w, 0x5410);
  o[3] = __byte_perm(v.y, v.w, 0x7632);
}
// Word j of lane c becomes word c of lane j, among four neighbouring lanes.
__device__ __forceinline__ void transpose4(uint4& v, int c) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int b = 1; b <= 2; b *= 2) {
    const bool up = c & b;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(i & b)) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[i] : w[i | b], b);
        if (up) w[i] = got;
        else w[i | b] = got;
      }
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
__device__ __forceinline__ __nv_bfloat162 offset_of(uint32_t z) {
  return as_pair(0x43004300u | z | z << 16);
}

// kM tiles of 16 weight rows and kN tiles of 8 tokens for every warp.  kFine: groups of 32 or 64 columns, so a product may not
// span a step: four lanes exchange their words and then hold neighbouring columns.
template <int kM, int kN, bool kFine> __global__ void __launch_bounds__(32 * kWarps) w4_few_kernel(const FewParams p) {
  __shared__ float sums[kWarps][kN * 8][kM * 16 + 1];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int tile = blockIdx.x / p.split, rank = blockIdx.x % p.split;
  const int row0 = tile * kM * 16, tok0 = blockIdx.y * kN * 8;
  const int steps = (p.K + kStep - 1) / kStep, stride = kWarps * p.split;
  const int groups = p.K / p.group;

  float acc[kM][kN][4], part[kM][kN][4];
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = part[m][n][i] = 0.f;

  uint4 next[kM][2];
  auto fetch = [&](int u) {
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0 + m * 16 + h * 8 + g;
        next[m][h] = make_uint4(0, 0, 0, 0);
        if (u < steps && row < p.N && u * kStep + c * 32 < p.K)
          next[m][h] = ptx::ld_nc_v4(p.q + (long long)row * (p.K / 2) + u * (kStep / 2) + c * 16);
      }
  };
  const int u0 = rank * kWarps + warp;
  fetch(u0);
  for (int u = u0; u < steps; u += stride) {
    uint4 w[kM][2];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[m][h] = next[m][h];
    fetch(u + stride);
    if constexpr (kFine) {
#pragma unroll
      for (int m = 0; m < kM; ++m) { transpose4(w[m][0], c); transpose4(w[m][1], c); }
    }
    __nv_bfloat162 off[kM][2];
    float scale[kM][2];
    auto group_of = [&](int k) {
      const int at = k / p.group;
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = row0 + m * 16 + h * 8 + g;
          const bool in = row < p.N && k < p.K;
          const long long i = (long long)row * groups + at;
          scale[m][h] = in ? __bfloat162float(p.s[i]) : 0.f;
          off[m][h] = offset_of(in && p.z ? p.z[i] : 8);
        }
    };
    if (!kFine) group_of(u * kStep);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int block = u * kStep + j * 32;            // kFine: the 32 columns that the four lanes hold now
      if (kFine && block % p.group == 0) group_of(block);
      uint32_t b[kN][4];
      const int k = kFine ? block + c * 8 : u * kStep + c * 32 + j * 8;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int tok = tok0 + n * 8 + g;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (tok < p.T && k < p.K) v = __ldg(reinterpret_cast<const uint4*>(p.x + (long long)tok * p.ldx + k));
        pair_up(v, b[n]);
      }
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        uint32_t lo[4], hi[4];
        widen(word(w[m][0], j), off[m][0], lo);
        widen(word(w[m][1], j), off[m][1], hi);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          mma(part[m][n], lo[0], hi[0], lo[1], hi[1], b[n][0], b[n][1]);
          mma(part[m][n], lo[2], hi[2], lo[3], hi[3], b[n][2], b[n][3]);
        }
      }
      if (j == 3 || (kFine && (block + 32) % p.group == 0)) {
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              acc[m][n][i] = fmaf(scale[m][i / 2], part[m][n][i], acc[m][n][i]);
              part[m][n][i] = 0.f;
            }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[warp][n * 8 + c * 2 + i % 2][m * 16 + i / 2 * 8 + g] = acc[m][n][i];
  __syncthreads();
  constexpr int kTile = kM * 16 * kN * 8;
  for (int e = threadIdx.x; e < kTile; e += 32 * kWarps) {
    const int r = e % (kM * 16), t = e / (kM * 16);
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += sums[i][t][r];
    sums[0][t][r] = v;                                // nobody else reads or writes this element's words
  }
  if (p.split > 1) {
    // the cluster's blocks add up their sums in the blocks' order, each for its share of the tile
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    for (int e = rank * 32 * kWarps + threadIdx.x; e < kTile; e += p.split * 32 * kWarps) {
      const int r = e % (kM * 16), t = e / (kM * 16);
      float v = 0.f;
      for (int i = 0; i < p.split; ++i) {
        uint32_t at;
        float f;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(ptx::smem_u32(&sums[0][t][r])), "r"(i));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at) : "memory");
        v += f;
      }
      if (tok0 + t < p.T && row0 + r < p.N) p.out[(tok0 + t) * p.ldo + row0 + r] = __float2bfloat16_rn(v);
    }
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");   // their memory stays until all have read
  } else {
    __syncthreads();
    for (int e = threadIdx.x; e < kTile; e += 32 * kWarps) {
      const int r = e % (kM * 16), t = e / (kM * 16);
      if (tok0 + t < p.T && row0 + r < p.N) p.out[(tok0 + t) * p.ldo + row0 + r] = __float2bfloat16_rn(sums[0][t][r]);
    }
  }
}

// w in bf16, for products with many tokens on the bf16 kernels: each weight is rounded once (2^-9 of itself at most), as a layer
// that keeps its weights in bf16 has them.  A thread has 32 columns, which are in one group.
struct WidenParams {
  const uint8_t* q;
  const __nv_bfloat16* s;
  const uint8_t* z;
  __nv_bfloat16* w;
  long long pieces;                                   // N * K / 32
  int K, group;
};
__global__ void __launch_bounds__(256) w4_widen_kernel(const WidenParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.pieces) return;
  const long long g = i * 32 / p.group;               // K is whole groups, so rows need no looking at
  const float s = __bfloat162float(p.s[g]), z = p.z ? (float)p.z[g] : 8.f;
  const uint4 v = ptx::ld_nc_v4(p.q + i * 16);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = word(v, j);
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = as_word(__floats2bfloat162_rn(((float)(w >> (8 * k) & 15) - z) * s, ((float)(w >> (8 * k + 4) & 15) - z) * s));
    }
    ptx::st_v4(p.w + i * 32 + j * 8, make_uint4(o[0], o[1], o[2], o[3]));
  }
}

// bf16 weights to 4 bits; a warp has a group.  Without zero points the scale is (largest magnitude) / 7, with them
// (largest - smallest) / 15 of a range that has zero in it, rounded to bf16; q is the nearest of what that can say.
struct QuantParams {
  const __nv_bfloat16* w;
  long long ldw;
  uint8_t* q;
  __nv_bfloat16* s;
  uint8_t* z;
  long long total;                                    // groups of the matrix
  int K, group;
};
__global__ void __launch_bounds__(256) w4_quant_kernel(const QuantParams p) {
  const long long i = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (i >= p.total) return;                           // a whole warp
  const long long per_row = p.K / p.group, row = i / per_row;
  const int k0 = (int)(i - row * per_row) * p.group;
  const __nv_bfloat16* w = p.w + row * p.ldw + k0;
  float lo = 0.f, hi = 0.f;
  for (int k = lane; k < p.group; k += 32) {
    const float v = __bfloat162float(w[k]);
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(p.z ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f));
  const float s = __bfloat162float(sb);
  const float z = !p.z ? 8.f : s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 0.f;
  if (lane == 0) {
    p.s[i] = sb;
    if (p.z) p.z[i] = (uint8_t)z;
  }
  for (int k = 2 * lane; k < p.group; k += 64) {
    uint32_t b = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float v = s > 0.f ? rintf(__fdiv_rn(__bfloat162float(w[k + h]), s)) + z : z;
      b |= (uint32_t)fminf(fmaxf(v, 0.f), 15.f) << (4 * h);
    }
    p.q[row * (p.K / 2) + (k0 + k) / 2] = (uint8_t)b;
  }
}

int sm_count(int* out) {
  static int counts[64];                              // racing threads write the same number
  int dev = 0;
  BSHMEM_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64) { host::last_error() = "w4: device number over 63"; return 1; }
  if (!counts[dev]) {
    int c = 0;
    BSHMEM_CUDA_TRY(cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev));
    counts[dev] = c;
  }
  *out = counts[dev];
  return 0;
}

template <typename K, typename P> int launch(K* kernel, dim3 grid, int threads, int cluster, const P& p, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  BSHMEM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return 0;
}

template <int kM, int kN> int few(FewParams& p, int sms, void* stream) {
  const int tiles = (p.N + kM * 16 - 1) / (kM * 16), tokens = (p.T + kN * 8 - 1) / (kN * 8), steps = (p.K + kStep - 1) / kStep;
  p.split = 1;
  while (p.split < 8 && (long long)tiles * tokens * p.split * 2 <= 3LL * sms && steps >= 2 * kWarps * p.split) p.split *= 2;
  const dim3 grid((unsigned)(tiles * p.split), (unsigned)tokens);
  if (p.group % kStep == 0) return launch(w4_few_kernel<kM, kN, false>, grid, 32 * kWarps, p.split, p, stream);
  return launch(w4_few_kernel<kM, kN, true>, grid, 32 * kWarps, p.split, p, stream);
}

bool aligned(const void* p) { return !(reinterpret_cast<uintptr_t>(p) & 15); }
bool shape_ok(long long N, int K, int group) {
  if (N >= 1 && N <= 0x3fffffff && K >= 32 && K <= 1 << 24 && (group == 32 || group == 64 || (group > 0 && group % 128 == 0)) && K % group == 0) return true;
  host::last_error() = "w4: needs groups of 32, 64 or a multiple of 128 columns and rows of whole groups";
  return false;
}

}  // namespace

extern "C" {

const char* bshmem_w4_last_error() { return host::last_error().c_str(); }

// x [T, K] bf16 with row pitch ldx (elements, % 8 == 0), out [T, N] bf16 contiguous; z may be null.
int bshmem_w4_few(const void* x, long long ldx, const void* q, const void* s, const void* z, void* out, int T, int N, int K, int group,
                  void* stream) {
  if (!shape_ok(N, K, group)) return 1;
  if (ldx % 8 || !aligned(x) || !aligned(q) || T > 65535 * 8) { host::last_error() = "w4: needs 16-byte aligned x and q, row pitch % 8 == 0"; return 1; }
  if (T <= 0) return 0;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  FewParams p = {static_cast<const __nv_bfloat16*>(x), static_cast<const uint8_t*>(q), static_cast<const __nv_bfloat16*>(s),
                 static_cast<const uint8_t*>(z), static_cast<__nv_bfloat16*>(out), ldx, N, T, N, K, group, 1};
  if (T <= 8) return few<1, 1>(p, sms, stream);
  if (T <= 16) return few<2, 2>(p, sms, stream);
  return few<2, 4>(p, sms, stream);
}

// w [N, K] bf16 contiguous and 16-byte aligned.
int bshmem_w4_widen(const void* q, const void* s, const void* z, void* w, int N, int K, int group, void* stream) {
  if (!shape_ok(N, K, group)) return 1;
  if (!aligned(q) || !aligned(w)) { host::last_error() = "w4: needs 16-byte aligned q and w"; return 1; }
  const WidenParams p = {static_cast<const uint8_t*>(q), static_cast<const __nv_bfloat16*>(s), static_cast<const uint8_t*>(z),
                         static_cast<__nv_bfloat16*>(w), (long long)N * (K / 32), K, group};
  if ((p.pieces + 255) / 256 > 0x7fffffffLL) { host::last_error() = "w4: matrix too large"; return 1; }
  return launch(w4_widen_kernel, dim3((unsigned)((p.pieces + 255) / 256)), 256, 1, p, stream);
}

// w [N, K] bf16 with row pitch ldw -> q, s and, unless z is null, z.
int bshmem_w4_quant(const void* w, long long ldw, void* q, void* s, void* z, int N, int K, int group, void* stream) {
  if (!shape_ok(N, K, group)) return 1;
  const QuantParams p = {static_cast<const __nv_bfloat16*>(w), ldw, static_cast<uint8_t*>(q), static_cast<__nv_bfloat16*>(s),
                         static_cast<uint8_t*>(z), (long long)N * (K / group), K, group};
  if ((p.total + 7) / 8 > 0x7fffffffLL) { host::last_error() = "w4: matrix too large"; return 1; }
  w4_quant_kernel<<<(unsigned)((p.total + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  BSHMEM_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // extern "C"
