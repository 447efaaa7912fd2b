// norm_kernels.cuh — RMS norms before and after a block, with the block's gate, its residual scale and the residual sum.
//
//   n(v) = v / sqrt(mean(v^2) + eps)
//   kPost     out = x + s * g * w1 * n(y)              y: what the block returned, x: the residual stream
//   kPre      h   = w2 * n(x)
//   kPostPre  both, with h = w2 * n(out): the end of one block and the start of the next
//
// g is absent, one value per column (a learned gate), per row or per element; s is one number.  Backward, with
// t = w2 * dh, nz = n(z), ny = n(y), r = 1 / sqrt(mean + eps) and means over the row:
//   dz  = dout + r2 * (t - nz * mean(t * nz))           gradient of out (of x: the same)
//   u   = s * g * w1 * dz;  dy = r1 * (u - ny * mean(u * ny))
//   dw2 = sum over rows of dh * nz;  with C = sum over rows of g' * dz * ny (g' the gate unless it is one per column):
//   dw1 = s * gcol * C,  dgcol = s * w1 * C,  drow gate = s * sum over columns of w1 * dz * ny,
//   delement gate = s * w1 * dz * ny,  ds = sum over everything of g * w1 * dz * ny
#pragma once
#include "../include/bshmem_types.h"
#include "ptx.cuh"
#include "row_values.cuh"
#include "tma_host.h"

namespace bshmem {
namespace norms {

using namespace rows;

enum Mode : int { kPre = 0, kPost = 1, kPostPre = 2 };
enum Gate : int { kNoGate = 0, kColumn = 1, kRow = 2, kElement = 3 };

// A [rows, columns] operand: address and row pitch in elements.
struct Mat { void* p; long long ld; };

struct Params {
  Mat y, x, out, h, gate;               // gate: per row or element (a row gate: one element per row, `ld` apart)
  const void *w1, *w2, *gcol;
  const void* scale; float scale_value; // scale: address of the number in memory (T or fp32), or null
  float eps;
  float *rstd1, *rstd2;                 // [rows], kept for the backward pass (null in inference)
  uint8_t *q1, *e1, *q2, *e2;           // y and z in 8 bits (null: not kept)
  long long ldq, lde;
  long long rows;
  int n;                                // columns
  int gate_kind;
  int w1_f32, w2_f32, gcol_f32, gate_f32, scale_f32;
};

struct BwdParams {
  Mat dout, dh, z, y, gate, dz, dy, dgate;
  const void *w1, *w2, *gcol;
  const void* scale; float scale_value;
  const float *rstd1, *rstd2;
  const uint8_t *q1, *e1, *q2, *e2;
  long long ldq, lde;
  float *part_w2, *part_c, *part_s;     // [groups, n], [groups, n], [groups]; null where nobody asks
  long long rows;
  int n;
  int gate_kind;
  int w1_f32, w2_f32, gcol_f32, gate_f32, scale_f32;
};

template <typename T> __device__ __forceinline__ float number(const void* p, int f32, float otherwise) {
  return !p ? otherwise : f32 ? *static_cast<const float*>(p) : to_float<T>(*static_cast<const T*>(p));
}
template <typename T> __device__ __forceinline__ T* row_of(const Mat& m, long long row) { return static_cast<T*>(m.p) + row * m.ld; }

// One row per blockDim.x threads, kChunks groups of eight columns for each: the row stays in registers between the sums, so
// memory is read once.
template <typename T, int kMode, int kChunks, bool kVec>
__global__ void __launch_bounds__(kChunks == 4 ? 512 : 1024) norm_fwd_kernel(const Params p) {
  __shared__ float words[2 * kMaxWarps];
  RowSum sum(words);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const int n = live ? p.n : 0;
  const float inv_n = 1.f / (float)p.n;
  float z[kChunks][8];
  if constexpr (kMode != kPre) {
    Raw8<T> ry[kChunks], rx[kChunks];
    const T *y = row_of<T>(p.y, live ? row : 0), *x = row_of<T>(p.x, live ? row : 0);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      ry[i] = load8<kVec>(y, col, n);
      rx[i] = load8<kVec>(x, col, n);
    }
    float scale = number<T>(p.scale, p.scale_f32, p.scale_value);
    if (p.gate_kind == kRow && live) scale *= p.gate_f32 ? row_of<float>(p.gate, row)[0] : to_float<T>(row_of<T>(p.gate, row)[0]);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float v[8];
      unpack(ry[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    }
    const float rstd = rsqrtf(fmaf(sum(ss), inv_n, p.eps));
    if (p.rstd1 && live && threadIdx.x == 0) p.rstd1[row] = rstd;
    const float f = scale * rstd;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      float v[8], w[8];
      unpack(ry[i], v);
      if (p.q1) {
        uint32_t e;
        const uint2 q = encode8<T>(v, e);
        if (col < n) {
          *reinterpret_cast<uint2*>(p.q1 + row * p.ldq + col) = q;
          if (col % 128 == 0) p.e1[row * p.lde + col / 128] = (uint8_t)e;
        }
      }
      vector8<kVec, T>(p.w1, p.w1_f32, col, n, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= w[j] * f;
      if (p.gate_kind == kColumn) {
        vector8<kVec, T>(p.gcol, p.gcol_f32, col, n, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= w[j];
      } else if (p.gate_kind == kElement && live) {
        if (p.gate_f32) unpack(load8<kVec>(row_of<float>(p.gate, row), col, n), w);
        else unpack(load8<kVec>(row_of<T>(p.gate, row), col, n), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= w[j];
      }
      unpack(rx[i], w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += w[j];
      const Raw8<T> o = pack<T>(v);
      store8<kVec>(row_of<T>(p.out, live ? row : 0), col, n, o);
      unpack(o, z[i]);                                // the next norm is one of the stored sum
    }
  } else {
    const T* x = row_of<T>(p.x, live ? row : 0);
    Raw8<T> rx[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) rx[i] = load8<kVec>(x, (threadIdx.x + i * blockDim.x) * 8, n);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) unpack(rx[i], z[i]);
  }
  if constexpr (kMode != kPost) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(z[i][j], z[i][j], ss);       // columns behind the last one are zero
    const float rstd = rsqrtf(fmaf(sum(ss), inv_n, p.eps));
    if (p.rstd2 && live && threadIdx.x == 0) p.rstd2[row] = rstd;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      if (p.q2) {
        uint32_t e;
        const uint2 q = encode8<T>(z[i], e);
        if (col < n) {
          *reinterpret_cast<uint2*>(p.q2 + row * p.ldq + col) = q;
          if (col % 128 == 0) p.e2[row * p.lde + col / 128] = (uint8_t)e;
        }
      }
      float w[8];
      vector8<kVec, T>(p.w2, p.w2_f32, col, n, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= z[i][j] * rstd;
      store8<kVec>(row_of<T>(p.h, live ? row : 0), col, n, pack<T>(w));
    }
  }
}

// Eight values of an operand that was kept as it was, or in 8 bits.
template <bool kKept8, bool kVec, typename T>
__device__ __forceinline__ void kept8(const Mat& m, const uint8_t* q, const uint8_t* e, long long ldq, long long lde, long long row,
                                      int col, int n, float (&v)[8]) {
  if constexpr (kKept8) {
    uint2 b = make_uint2(0, 0);
    uint32_t x = 1;
    if (col < n) {
      b = __ldg(reinterpret_cast<const uint2*>(q + row * ldq + col));
      x = __ldg(e + row * lde + col / 128);
    }
    decode8(b, x, v);
  } else {
    unpack(load8<kVec>(row_of<T>(m, row), col, n), v);
  }
}

// A block walks over rows and keeps the column sums of its rows in registers; norm_bwd_finish_kernel adds up the groups' sums in
// their order, so two calls give the same bits.
template <typename T, int kMode, int kChunks, bool kVec, bool kKept8>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const BwdParams p) {
  __shared__ float words[2 * kMaxWarps];
  RowSum sum(words);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const float inv_n = 1.f / (float)p.n;
  const float scale = number<T>(p.scale, p.scale_f32, p.scale_value);
  float acc_w2[kMode != kPost ? kChunks : 1][8], acc_c[kMode != kPre ? kChunks : 1][8], acc_s = 0.f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kMode != kPost) acc_w2[i][j] = 0.f;
      if constexpr (kMode != kPre) acc_c[i][j] = 0.f;
    }
  const long long step = (long long)gridDim.x * blockDim.y;
  for (long long first = (long long)blockIdx.x * blockDim.y; first < p.rows; first += step) {      // the same for the whole block
    const bool live = first + threadIdx.y < p.rows;
    const long long row = live ? first + threadIdx.y : 0;
    const int n = live ? p.n : 0;
    float dz[kChunks][8], ny[kMode != kPre ? kChunks : 1][8];
    if constexpr (kMode != kPre) {
      const float rstd = __ldg(p.rstd1 + row);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        kept8<kKept8, kVec, T>(p.y, p.q1, p.e1, p.ldq, p.lde, row, col, n, ny[i]);
        if (p.dout.p) {
          unpack(load8<kVec>(row_of<T>(p.dout, row), col, n), dz[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) dz[i][j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ny[i][j] *= rstd;
      }
    }
    if constexpr (kMode != kPost) {
      float nz[kChunks][8], t[kChunks][8], dot = 0.f;
      const float rstd = __ldg(p.rstd2 + row);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        kept8<kKept8, kVec, T>(p.z, p.q2, p.e2, p.ldq, p.lde, row, col, n, nz[i]);
        unpack(load8<kVec>(row_of<T>(p.dh, row), col, n), t[i]);
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        float w[8];
        vector8<kVec, T>(p.w2, p.w2_f32, (threadIdx.x + i * blockDim.x) * 8, n, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          nz[i][j] *= rstd;
          acc_w2[i][j] = fmaf(t[i][j], nz[i][j], acc_w2[i][j]);
          t[i][j] *= w[j];
          dot = fmaf(t[i][j], nz[i][j], dot);
        }
      }
      const float mean = sum(dot) * inv_n;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = rstd * (t[i][j] - nz[i][j] * mean);
          if constexpr (kMode == kPre) dz[i][j] = d;
          else dz[i][j] += d;
        }
        store8<kVec>(row_of<T>(p.dz, row), (threadIdx.x + i * blockDim.x) * 8, n, pack<T>(dz[i]));
      }
    }
    if constexpr (kMode != kPre) {
      // v = dz * g * w1 without the row's gate and the scale; its sum with ny gives both of the scalar gradients and dy's mean
      float row_gate = 1.f;
      if (p.gate_kind == kRow && live) row_gate = p.gate_f32 ? row_of<float>(p.gate, row)[0] : to_float<T>(row_of<T>(p.gate, row)[0]);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        float w[8], g[8];
        vector8<kVec, T>(p.w1, p.w1_f32, col, n, w);
        if (p.gate_kind == kElement) {
          if (p.gate_f32) unpack(load8<kVec>(row_of<float>(p.gate, row), col, n), g);
          else unpack(load8<kVec>(row_of<T>(p.gate, row), col, n), g);
          if (p.dgate.p) {
            float d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = scale * w[j] * dz[i][j] * ny[i][j];
            if (p.gate_f32) store8<kVec>(row_of<float>(p.dgate, row), col, n, pack<float>(d));
            else store8<kVec>(row_of<T>(p.dgate, row), col, n, pack<T>(d));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            dz[i][j] *= g[j];
            acc_c[i][j] = fmaf(dz[i][j], ny[i][j], acc_c[i][j]);
            dz[i][j] *= w[j];
          }
        } else {
          if (p.gate_kind == kColumn) {
            vector8<kVec, T>(p.gcol, p.gcol_f32, col, n, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] *= g[j];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc_c[i][j] = fmaf(dz[i][j] * row_gate, ny[i][j], acc_c[i][j]);
            dz[i][j] *= w[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(dz[i][j], ny[i][j], dot);
      }
      dot = sum(dot);
      if (live) acc_s = fmaf(row_gate, dot, acc_s);
      if (p.gate_kind == kRow && p.dgate.p && live && threadIdx.x == 0) {
        if (p.gate_f32) row_of<float>(p.dgate, row)[0] = scale * dot;
        else row_of<T>(p.dgate, row)[0] = from_float<T>(scale * dot);
      }
      if (p.dy.p) {
        const float f = __ldg(p.rstd1 + row) * scale * row_gate, mean = dot * inv_n;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          float d[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] = f * (dz[i][j] - ny[i][j] * mean);
          store8<kVec>(row_of<T>(p.dy, row), (threadIdx.x + i * blockDim.x) * 8, n, pack<T>(d));
        }
      }
    }
  }
  const long long group = (long long)blockIdx.x * blockDim.y + threadIdx.y;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (threadIdx.x + i * blockDim.x) * 8;
    // part rows are padded to a multiple of eight columns by their pitch
    const long long at = group * ((p.n + 7) / 8 * 8) + col;
    if (col < p.n) {
      if constexpr (kMode != kPost)
        if (p.part_w2) {
          float4* o = reinterpret_cast<float4*>(p.part_w2 + at);
          o[0] = make_float4(acc_w2[i][0], acc_w2[i][1], acc_w2[i][2], acc_w2[i][3]);
          o[1] = make_float4(acc_w2[i][4], acc_w2[i][5], acc_w2[i][6], acc_w2[i][7]);
        }
      if constexpr (kMode != kPre)
        if (p.part_c) {
          float4* o = reinterpret_cast<float4*>(p.part_c + at);
          o[0] = make_float4(acc_c[i][0], acc_c[i][1], acc_c[i][2], acc_c[i][3]);
          o[1] = make_float4(acc_c[i][4], acc_c[i][5], acc_c[i][6], acc_c[i][7]);
        }
    }
  }
  if (kMode != kPre && p.part_s && threadIdx.x == 0) p.part_s[group] = acc_s;
}

// Threads of a row, rows of a block and eights of columns per thread for rows of n columns.
struct Shape { int threads, rows, chunks; };
constexpr int kMaxColumns = 16384;

inline int sm_count(int* out) {
  static int counts[64];                                       // racing threads write the same number
  int dev = 0;
  BSHMEM_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64) { host::last_error() = "norm: device number over 63"; return 1; }
  if (!counts[dev]) {
    int c = 0;
    BSHMEM_CUDA_TRY(cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev));
    counts[dev] = c;
  }
  *out = counts[dev];
  return 0;
}

template <typename K, typename P> int launch(K* kernel, dim3 grid, dim3 block, const P& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSHMEM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return 0;
}

inline Shape forward_shape(long long rows, int n, bool vec, int sms) {
  const int eights = (n + 7) / 8;
  // few rows: as many threads for each as it has eights; many: four eights per thread, whose loads are all on their way at once
  int chunks = !vec || rows > 2LL * sms ? 4 : 1;
  while (chunks < 4 && eights > 1024 * chunks) chunks *= 2;
  int threads = ((eights + chunks - 1) / chunks + 31) / 32 * 32;
  int per_block = threads >= 128 ? 1 : 128 / threads;
  if (per_block > rows) per_block = rows < 1 ? 1 : (int)rows;
  return {threads, per_block, chunks};
}
inline Shape backward_shape(long long rows, int n) {
  const int eights = (n + 7) / 8;
  const int chunks = eights > 1024 ? 4 : eights > 512 ? 2 : 1;
  const int threads = ((eights + chunks - 1) / chunks + 31) / 32 * 32;
  int per_block = threads >= 256 ? 1 : 256 / threads;
  if (per_block > rows) per_block = rows < 1 ? 1 : (int)rows;
  return {threads, per_block, chunks};
}

template <typename T, int kMode> int forward_mode(bool vec, const Params& p, cudaStream_t stream) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const Shape s = forward_shape(p.rows, p.n, vec, sms);
  const dim3 grid((unsigned)((p.rows + s.rows - 1) / s.rows)), block(s.threads, s.rows);
  if (!vec) return launch(norm_fwd_kernel<T, kMode, 4, false>, grid, block, p, stream);
  if (s.chunks == 1) return launch(norm_fwd_kernel<T, kMode, 1, true>, grid, block, p, stream);
  if (s.chunks == 2) return launch(norm_fwd_kernel<T, kMode, 2, true>, grid, block, p, stream);
  return launch(norm_fwd_kernel<T, kMode, 4, true>, grid, block, p, stream);
}
template <typename T, int kMode, bool kVec, bool kKept> int backward_form(int blocks, const BwdParams& p, cudaStream_t stream) {
  const Shape s = backward_shape(p.rows, p.n);
  const dim3 grid((unsigned)blocks), block(s.threads, s.rows);
  if (s.chunks == 1) return launch(norm_bwd_kernel<T, kMode, 1, kVec, kKept>, grid, block, p, stream);
  if (s.chunks == 2) return launch(norm_bwd_kernel<T, kMode, 2, kVec, kKept>, grid, block, p, stream);
  return launch(norm_bwd_kernel<T, kMode, 4, kVec, kKept>, grid, block, p, stream);
}
template <typename T, int kMode> int backward_mode(bool vec, bool kept, int blocks, const BwdParams& p, cudaStream_t stream) {
  if (vec) return kept ? backward_form<T, kMode, true, true>(blocks, p, stream) : backward_form<T, kMode, true, false>(blocks, p, stream);
  return kept ? backward_form<T, kMode, false, true>(blocks, p, stream) : backward_form<T, kMode, false, false>(blocks, p, stream);
}

// The kernels for one type of rows; norm_bf16.cu, norm_fp16.cu and norm_fp32.cu instantiate them.
template <typename T> int forward(int mode, bool vec, const Params& p, cudaStream_t stream) {
  return mode == kPre ? forward_mode<T, kPre>(vec, p, stream) : mode == kPost ? forward_mode<T, kPost>(vec, p, stream)
                                                                              : forward_mode<T, kPostPre>(vec, p, stream);
}
template <typename T> int backward(int mode, bool vec, bool kept, int blocks, const BwdParams& p, cudaStream_t stream) {
  return mode == kPre ? backward_mode<T, kPre>(vec, kept, blocks, p, stream)
         : mode == kPost ? backward_mode<T, kPost>(vec, kept, blocks, p, stream) : backward_mode<T, kPostPre>(vec, kept, blocks, p, stream);
}

}  // namespace norms
}  // namespace bshmem
