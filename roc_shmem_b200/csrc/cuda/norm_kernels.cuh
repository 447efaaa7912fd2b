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
  uint8_t* end; int tail;               // bytes behind the last exponent, up to a whole word: zeros
  long long ldq, lde;
  long long rows;
  int n;                                // columns
  int gate_kind;
  int w1_f32, w2_f32, gcol_f32, gate_f32, scale_f32;
  int stages, ring_words;               // see Ring
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
  int stages, ring_words;
  int held;                             // the weights are in shared memory: 1 in fp32, 2 as they are (see backward_raw)
};

template <typename T> __device__ __forceinline__ float number(const void* p, int f32, float otherwise) {
  return !p ? otherwise : f32 ? *static_cast<const float*>(p) : to_float<T>(*static_cast<const T*>(p));
}
template <typename T> __device__ __forceinline__ T* row_of(const Mat& m, long long row) { return static_cast<T*>(m.p) + row * m.ld; }

// How a kernel gets its rows.  kScalar: value by value, for rows off 16-byte boundaries or of odd sizes.  kDirect: 16-byte loads into
// registers.  kRing: a block walks over rows, and each thread has the next rows' words that it will need itself on their way into
// shared memory (cp.async), so nothing but its own wait is between the copy and the use.
enum Form : int { kScalar = 0, kDirect = 1, kRing = 2 };

// What is known of a gate per element when a kernel is built: that there is none, that it has the rows' type, that it is fp32, or nothing.
enum Element : int { kNone = 0, kOfT = 1, kOfF32 = 2, kAsk = 3 };
template <int kElement> __device__ __forceinline__ bool element_gate(int gate_kind) { return kElement == kAsk ? gate_kind == Gate::kElement : kElement != kNone; }
template <int kElement> __device__ __forceinline__ bool element_f32(int gate_f32) { return kElement == kAsk ? gate_f32 : kElement == kOfF32; }

__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// Through L1: the two halves of a sector of fp32 come with two copies, and the second finds it there.  One norm of 16384 x 4096 in fp32 takes
// 103 us so, 129 past L1.
__device__ __forceinline__ void cp_async_16_near(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// The words of a thread in one stage of the ring, [stage][word][thread].  A thread reads what it copied itself.
struct Ring {
  uint4* mine;
  int words, threads, stages;
  __device__ __forceinline__ Ring(uint4* base, int w, int s) : words(w), threads(blockDim.x * blockDim.y), stages(s) {
    mine = base + threadIdx.y * blockDim.x + threadIdx.x;
  }
  __device__ __forceinline__ uint4* at(int stage, int word) const { return mine + (stage * words + word) * threads; }
  __device__ __forceinline__ void clear(int stage) const {
    for (int i = 0; i < words; ++i) *at(stage, i) = make_uint4(0, 0, 0, 0);
  }
  // The oldest of `stages` rows on their way has arrived.
  __device__ __forceinline__ void wait() const {
    if (stages == 2) ptx::cp_async_wait<1>();
    else ptx::cp_async_wait<2>();
  }
  template <typename T> __device__ __forceinline__ void fetch8(int stage, int word, const T* from) const {
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords; ++i) {
      const uint32_t to = ptx::smem_u32(at(stage, word + i));
      if constexpr (Raw8<T>::kWords == 1) ptx::cp_async_16(to, from);
      else cp_async_16_near(to, reinterpret_cast<const uint4*>(from) + i);
    }
  }
  template <typename T> __device__ __forceinline__ Vals get8(int stage, int word) const {
    Raw8<T> v;
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords; ++i) v.set(i, *at(stage, word + i));
    return unpack(v);
  }
};
__device__ __forceinline__ float sum2(float2 v) { return v.x + v.y; }

// ---- forward -------------------------------------------------------------------------------------------
// Threads of a multiprocessor for rows in a ring.  1024 have 64 registers each, which holds two eights of a row and of its weights: 16384 x
// 4096 before a block 47 us.  `more` (8 bits or a gate per element) with both norms does not fit: 8192 x 8192 with a gate per
// element takes 109 us with 512, 118 with 1024; one norm with 8 bits, 16384 x 4096 with its gradient, 231 with 512, 176 with 1024.
constexpr int ring_threads(int mode, int chunks, bool more) { return chunks > 2 || (mode == kPostPre && more) ? 512 : 1024; }
// A row stays in the registers of its threads, kChunks groups of eight columns for each, between the sums: memory is read once.
// In a ring the weights (w1 times a gate per column, and w2) stay in registers too, and whether the inputs are kept in 8 bits (kKeep) and
// what gate per element there is are known when the kernel is built: 8192 x 8192 with neither takes 95 us so, 110 where the kernel asks at
// every row.  In the other forms it asks.
template <typename T, int kMode, int kChunks, int kForm, bool kKeep = true, int kElement = kAsk>
__global__ void __launch_bounds__(kForm == kRing ? ring_threads(kMode, kChunks, kKeep || kElement != kNone) : kForm == kDirect && kChunks == 1 ? 1024 : 512)
    norm_fwd_kernel(const Params p) {
  constexpr int kAccess = kForm == kScalar ? kStrided : kVector;
  constexpr bool kHeld = kForm == kRing && kChunks <= 2;
  constexpr int W = Raw8<T>::kWords, kX = kMode == kPre ? 0 : kChunks * W, kGate = kX + kChunks * W;
  extern __shared__ uint4 ring_words[];
  __shared__ float sums[2 * kMaxWarps];
  RowSum sum(sums);
  const bool keep = kForm == kRing ? kKeep : p.q1 || p.q2, per_element = kMode != kPre && element_gate<kElement>(p.gate_kind);
  const bool f32 = element_f32<kElement>(p.gate_f32);
  const Ring ring(ring_words, p.ring_words, p.stages);
  if constexpr (kForm == kRing) {
    for (int i = 0; i < p.stages; ++i) ring.clear(i);        // columns behind the last one are never fetched
    __syncthreads();
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (keep && blockIdx.x == 0 && threadIdx.y == 0 && threadIdx.x < p.tail) p.end[threadIdx.x] = 0;
  const float inv_n = 1.f / (float)p.n;
  const long long step = (long long)gridDim.x * blockDim.y;
  auto column = [&](int i) { return (int)(threadIdx.x + i * blockDim.x) * 8; };
  auto fetch = [&](long long row, int stage) {
    if (row < p.rows) {
      const T *y = row_of<T>(p.y, row), *x = row_of<T>(p.x, row);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = column(i);
        if (col < p.n) {
          if constexpr (kMode != kPre) ring.fetch8(stage, i * W, y + col);
          ring.fetch8(stage, kX + i * W, x + col);
          if (per_element) {
            if (f32) ring.fetch8(stage, kGate + i * 2, row_of<float>(p.gate, row) + col);
            else ring.fetch8(stage, kGate + i * W, row_of<T>(p.gate, row) + col);
          }
        }
      }
    } else {
      ring.clear(stage);
    }
    ptx::cp_async_commit();
  };
  long long first = (long long)blockIdx.x * blockDim.y;
  int stage = 0;
  if constexpr (kForm == kRing)
    for (int i = 0; i < p.stages; ++i) fetch(first + threadIdx.y + i * step, i);
  const float scale0 = number<T>(p.scale, p.scale_f32, p.scale_value);
  auto weight1 = [&](int i) {
    Vals w = vector8<kAccess, T>(p.w1, p.w1_f32, column(i), p.n);
    if (p.gate_kind == kColumn) {
      const Vals g = vector8<kAccess, T>(p.gcol, p.gcol_f32, column(i), p.n);
#pragma unroll
      for (int j = 0; j < 4; ++j) w.p[j] = mul2(w.p[j], g.p[j]);
    }
    return w;
  };
  Vals held1[kHeld ? kChunks : 1], held2[kHeld ? kChunks : 1];
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if constexpr (kMode != kPre) held1[i] = weight1(i);
      if constexpr (kMode != kPost) held2[i] = vector8<kAccess, T>(p.w2, p.w2_f32, column(i), p.n);
    }
  }
  for (; first < p.rows; first += step) {                    // the same for the whole block
    const bool live = first + threadIdx.y < p.rows;
    const long long row = live ? first + threadIdx.y : 0;
    const int n = live ? p.n : 0;
    if constexpr (kForm == kRing) ring.wait();
    Vals z[kChunks];
    if constexpr (kMode != kPre) {
      Vals y[kChunks], x[kForm == kRing ? 1 : kChunks];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (kForm == kRing) {
          y[i] = ring.get8<T>(stage, i * W);
        } else {
          y[i] = unpack(load8<kAccess>(row_of<T>(p.y, row), column(i), n));
          x[i] = unpack(load8<kAccess>(row_of<T>(p.x, row), column(i), n));
        }
      }
      float scale = scale0;
      if (p.gate_kind == kRow && live) scale *= p.gate_f32 ? row_of<float>(p.gate, row)[0] : to_float<T>(row_of<T>(p.gate, row)[0]);
      float2 ss = both(0.f);
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fma2(y[i].p[j], y[i].p[j], ss);
      const float rstd = rsqrtf(fmaf(sum(sum2(ss)), inv_n, p.eps));
      if (p.rstd1 && live && threadIdx.x == 0) p.rstd1[row] = rstd;
      const float2 f = both(scale * rstd);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = column(i);
        if (keep) keep8<kAccess, T>(p.q1 + row * p.ldq, p.e1 + row * p.lde, col, n, y[i]);
        Vals w, r;
        if constexpr (kHeld) w = held1[i];
        else w = weight1(i);
        if constexpr (kForm == kRing) r = ring.get8<T>(stage, kX + i * W);
        else r = x[i];
        if (per_element) {
          Vals g;
          if constexpr (kForm == kRing) g = f32 ? ring.get8<float>(stage, kGate + i * 2) : ring.get8<T>(stage, kGate + i * W);
          else g = f32 ? unpack(load8<kAccess>(row_of<float>(p.gate, row), col, n)) : unpack(load8<kAccess>(row_of<T>(p.gate, row), col, n));
#pragma unroll
          for (int j = 0; j < 4; ++j) w.p[j] = mul2(w.p[j], g.p[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) r.p[j] = fma2(mul2(y[i].p[j], f), w.p[j], r.p[j]);
        const Raw8<T> o = pack<T>(r);
        store8<kAccess>(row_of<T>(p.out, row), col, n, o);
        if constexpr (kMode == kPostPre) z[i] = unpack(o);   // the next norm is one of the stored sum
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (kForm == kRing) z[i] = ring.get8<T>(stage, i * W);
        else z[i] = unpack(load8<kAccess>(row_of<T>(p.x, row), column(i), n));
      }
    }
    if constexpr (kForm == kRing) {
      fetch(first + threadIdx.y + p.stages * step, stage);   // this thread has read its words of the stage
      if (++stage == p.stages) stage = 0;
    }
    if constexpr (kMode != kPost) {
      float2 ss = both(0.f);
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fma2(z[i].p[j], z[i].p[j], ss);   // columns behind the last one are zero
      const float rstd = rsqrtf(fmaf(sum(sum2(ss)), inv_n, p.eps));
      if (p.rstd2 && live && threadIdx.x == 0) p.rstd2[row] = rstd;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = column(i);
        if (keep) keep8<kAccess, T>(p.q2 + row * p.ldq, p.e2 + row * p.lde, col, n, z[i]);
        Vals w;
        if constexpr (kHeld) w = held2[i];
        else w = vector8<kAccess, T>(p.w2, p.w2_f32, col, n);
#pragma unroll
        for (int j = 0; j < 4; ++j) w.p[j] = mul2(mul2(z[i].p[j], both(rstd)), w.p[j]);
        store8<kAccess>(row_of<T>(p.h, row), col, n, pack<T>(w));
      }
    }
  }
}

// ---- backward ------------------------------------------------------------------------------------------
// A block walks over rows and keeps the column sums of its rows in registers; norm_bwd_finish_kernel adds up the groups' sums in
// their order, so two calls give the same bits.  In a ring the weights are fp32 words of shared memory behind the stages, where
// there is room.  kLong: rows of over 8192 columns on 1024 threads, whose 64 registers do not hold the column sums: words of shared
// memory do, which only their thread touches.  kHeld: the usual call of a ring, known when the kernel is built: the weights are held (1, 2: see
// BwdParams), dout is there, dy is wanted, and what gate per element there is; 0: the kernel asks.  8192 x 8192 with its forward pass 243 us
// for 251, 16384 x 4096 with 8 bits and a gate per element 379 for 397.
template <typename T, int kMode, int kChunks, int kForm, bool kKept8, int kHeld = 0, int kElement = kAsk, bool kLong = false>
__global__ void __launch_bounds__(kLong ? 1024 : 512) norm_bwd_kernel(const BwdParams p) {
  constexpr int kAccess = kForm == kScalar ? kStrided : kVector;
  // words of a stage: dout, dh, z, y, the two 1 / sqrt(...) and the gate per element; one that is kept in 8 bits has its
  // eight bytes and the four that its exponent byte is among in one word
  constexpr int W = Raw8<T>::kWords, K = kKept8 ? 1 : W;
  constexpr int kDh = kMode == kPre ? 0 : kChunks * W, kZ = kDh + (kMode == kPost ? 0 : kChunks * W);
  constexpr int kY = kZ + (kMode == kPost ? 0 : kChunks * K), kRstd = kY + (kMode == kPre ? 0 : kChunks * K), kGate = kRstd + 1;
  constexpr int kW2 = kMode == kPre ? 0 : kChunks * 2;       // words of the weights: w1 times a gate per column, w2
  extern __shared__ uint4 ring_words[];
  __shared__ float sums[2 * kMaxWarps];
  RowSum sum(sums);
  const bool per_element = kMode != kPre && element_gate<kElement>(p.gate_kind), f32 = element_f32<kElement>(p.gate_f32);
  const bool has_dout = kHeld || p.dout.p, wants_dy = kHeld || p.dy.p;
  const bool in_fp32 = kHeld ? kHeld == 1 : p.held == 1;
  const Ring ring(ring_words, p.ring_words, p.stages);
  const Ring weights(ring_words + p.stages * p.ring_words * ring.threads, 0, 0);
  if constexpr (kForm == kRing) {
    for (int i = 0; i < p.stages; ++i) ring.clear(i);
    __syncthreads();
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const float inv_n = 1.f / (float)p.n;
  const float scale = number<T>(p.scale, p.scale_f32, p.scale_value);
  Vals acc_w2[kMode != kPost && !kLong ? kChunks : 1], acc_c[kMode != kPre && !kLong ? kChunks : 1];
  float acc_s = 0.f;
  const Ring accs(ring_words, 0, 0);                         // kLong: [sum][thread]
  auto hold = [](const Ring& r, int word, const Vals& v) {
    r.mine[word * r.threads] = make_uint4(__float_as_uint(v.p[0].x), __float_as_uint(v.p[0].y), __float_as_uint(v.p[1].x), __float_as_uint(v.p[1].y));
    r.mine[(word + 1) * r.threads] = make_uint4(__float_as_uint(v.p[2].x), __float_as_uint(v.p[2].y), __float_as_uint(v.p[3].x), __float_as_uint(v.p[3].y));
  };
  constexpr int kAccC = kMode == kPost ? 0 : kChunks * 2;    // words of the first sum, of w2
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    Vals zero;
    zero.fill(0.f);
    if constexpr (kLong) {
      if constexpr (kMode != kPost) hold(accs, i * 2, zero);
      if constexpr (kMode != kPre) hold(accs, kAccC + i * 2, zero);
    } else {
      if constexpr (kMode != kPost) acc_w2[i] = zero;
      if constexpr (kMode != kPre) acc_c[i] = zero;
    }
  }
  const long long step = (long long)gridDim.x * blockDim.y;
  auto column = [&](int i) { return (int)(threadIdx.x + i * blockDim.x) * 8; };
  auto fetch_kept = [&](int stage, int word, const Mat& m, const uint8_t* q, const uint8_t* e, long long row, int col) {
    if constexpr (kKept8) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(e + row * p.lde + col / 128);
      const uint32_t slot = ptx::smem_u32(ring.at(stage, word));
      cp_async_8(slot, q + row * p.ldq + col);
      ptx::cp_async_4(slot + 8, reinterpret_cast<const void*>(at & ~(uintptr_t)3));
    } else {
      ring.fetch8(stage, word, row_of<T>(m, row) + col);
    }
  };
  auto kept = [&](int stage, int word, const Mat& m, const uint8_t* q, const uint8_t* e, long long row, int col, int n) {
    if constexpr (kForm == kRing && kKept8) {
      const uint4 w = *ring.at(stage, word);
      const uint32_t byte = (uint32_t)reinterpret_cast<uintptr_t>(e + row * p.lde + col / 128) & 3;
      return decode8(make_uint2(w.x, w.y), w.z >> (8 * byte) & 255);
    } else if constexpr (kForm == kRing) {
      return ring.get8<T>(stage, word);
    } else if constexpr (kKept8) {
      return kept8<kAccess>(q + row * p.ldq, e + row * p.lde, col, n);
    } else {
      return unpack(load8<kAccess>(row_of<T>(m, row), col, n));
    }
  };
  auto plain = [&](int stage, int word, const Mat& m, long long row, int col, int n) {
    if constexpr (kForm == kRing) return ring.get8<T>(stage, word);
    else return unpack(load8<kAccess>(row_of<T>(m, row), col, n));
  };
  auto fetch = [&](long long row, int stage) {
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = column(i);
        if (col < p.n) {
          if constexpr (kMode != kPre) {
            if (has_dout) ring.fetch8(stage, i * W, row_of<T>(p.dout, row) + col);
            fetch_kept(stage, kY + i * K, p.y, p.q1, p.e1, row, col);
            if (per_element) {
              if (f32) ring.fetch8(stage, kGate + i * 2, row_of<float>(p.gate, row) + col);
              else ring.fetch8(stage, kGate + i * W, row_of<T>(p.gate, row) + col);
            }
          }
          if constexpr (kMode != kPost) {
            ring.fetch8(stage, kDh + i * W, row_of<T>(p.dh, row) + col);
            fetch_kept(stage, kZ + i * K, p.z, p.q2, p.e2, row, col);
          }
        }
      }
      const uint32_t slot = ptx::smem_u32(ring.at(stage, kRstd));
      if constexpr (kMode != kPre) ptx::cp_async_4(slot, p.rstd1 + row);
      if constexpr (kMode != kPost) ptx::cp_async_4(slot + 4, p.rstd2 + row);
    } else {
      ring.clear(stage);
    }
    ptx::cp_async_commit();
  };
  long long first = (long long)blockIdx.x * blockDim.y;
  int stage = 0;
  auto weight1 = [&](int i, int n) {
    Vals w = vector8<kAccess, T>(p.w1, p.w1_f32, column(i), n);
    if (p.gate_kind == kColumn) {
      const Vals g = vector8<kAccess, T>(p.gcol, p.gcol_f32, column(i), n);
#pragma unroll
      for (int j = 0; j < 4; ++j) w.p[j] = mul2(w.p[j], g.p[j]);
    }
    return w;
  };
  auto keep = [&](int i, int from, const Vals& v) {
    if (in_fp32) hold(weights, from + i * 2, v);
    else weights.mine[(from / 2 + i) * weights.threads] = pack<T>(v).get(0);
  };
  auto held = [&](int i, int from) { return in_fp32 ? weights.get8<float>(0, from + i * 2) : weights.get8<T>(0, from / 2 + i); };
  if constexpr (kForm == kRing) {
    for (int i = 0; i < p.stages; ++i) fetch(first + threadIdx.y + i * step, i);
    if (kHeld || p.held) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (kMode != kPre) keep(i, 0, weight1(i, p.n));
        if constexpr (kMode != kPost) keep(i, kW2, vector8<kAccess, T>(p.w2, p.w2_f32, column(i), p.n));
      }
    }
  }
  for (; first < p.rows; first += step) {                    // the same for the whole block
    const bool live = first + threadIdx.y < p.rows;
    const long long row = live ? first + threadIdx.y : 0;
    const int n = live ? p.n : 0;
    float row_gate = 1.f;
    if (kMode != kPre && p.gate_kind == kRow && live)
      row_gate = p.gate_f32 ? row_of<float>(p.gate, row)[0] : to_float<T>(row_of<T>(p.gate, row)[0]);
    float rstd1 = 0.f, rstd2 = 0.f;
    if constexpr (kForm == kRing) {
      ring.wait();
      const uint4 r = *ring.at(stage, kRstd);
      rstd1 = __uint_as_float(r.x);
      rstd2 = __uint_as_float(r.y);
    } else {
      if constexpr (kMode != kPre) rstd1 = p.rstd1[row];
      if constexpr (kMode != kPost) rstd2 = p.rstd2[row];
    }
    Vals dz[kChunks], ny[kMode != kPre ? kChunks : 1];
    // in a ring the first norm's operands are read when it is their turn; elsewhere their loads begin here
    auto first_norm = [&](int i) {
      ny[i] = kept(stage, kY + i * K, p.y, p.q1, p.e1, row, column(i), n);
#pragma unroll
      for (int j = 0; j < 4; ++j) ny[i].p[j] = mul2(ny[i].p[j], both(rstd1));
    };
    auto given = [&](int i) {
      if (has_dout) dz[i] = plain(stage, i * W, p.dout, row, column(i), n);
      else dz[i].fill(0.f);
    };
    if constexpr (kMode == kPost || (kMode == kPostPre && kForm != kRing)) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) { first_norm(i); given(i); }
    }
    if constexpr (kMode != kPost) {
      Vals nz[kChunks], t[kChunks];
      float2 dot = both(0.f);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        nz[i] = kept(stage, kZ + i * K, p.z, p.q2, p.e2, row, column(i), n);
        t[i] = plain(stage, kDh + i * W, p.dh, row, column(i), n);
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        Vals w;
        if (kForm == kRing && (kHeld || p.held)) w = held(i, kW2);
        else w = vector8<kAccess, T>(p.w2, p.w2_f32, column(i), n);
        Vals sums_w2;
        if constexpr (kLong) sums_w2 = accs.get8<float>(0, i * 2);
        else sums_w2 = acc_w2[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          nz[i].p[j] = mul2(nz[i].p[j], both(rstd2));
          sums_w2.p[j] = fma2(t[i].p[j], nz[i].p[j], sums_w2.p[j]);
          t[i].p[j] = mul2(t[i].p[j], w.p[j]);
          dot = fma2(t[i].p[j], nz[i].p[j], dot);
        }
        if constexpr (kLong) hold(accs, i * 2, sums_w2);
        else acc_w2[i] = sums_w2;
      }
      const float mean = sum(sum2(dot)) * inv_n;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (kMode == kPostPre && kForm == kRing) given(i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 d = fma2(nz[i].p[j], both(-mean), t[i].p[j]);
          if constexpr (kMode == kPre) dz[i].p[j] = mul2(d, both(rstd2));
          else dz[i].p[j] = fma2(d, both(rstd2), dz[i].p[j]);
        }
        store8<kAccess>(row_of<T>(p.dz, row), column(i), n, pack<T>(dz[i]));
      }
    }
    if constexpr (kMode != kPre) {
      // v = dz * g * w1 without the row's gate and the scale; its sum with ny gives both of the scalar gradients and dy's mean
      float2 dot2 = both(0.f);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = column(i);
        if constexpr (kMode == kPostPre && kForm == kRing) first_norm(i);
        Vals w;
        if (kForm == kRing && (kHeld || p.held)) w = held(i, 0);
        else w = weight1(i, n);
        if (per_element) {
          Vals g;
          if constexpr (kForm == kRing) g = f32 ? ring.get8<float>(stage, kGate + i * 2) : ring.get8<T>(stage, kGate + i * W);
          else g = f32 ? unpack(load8<kAccess>(row_of<float>(p.gate, row), col, n)) : unpack(load8<kAccess>(row_of<T>(p.gate, row), col, n));
          if (p.dgate.p) {
            Vals d;
#pragma unroll
            for (int j = 0; j < 4; ++j) d.p[j] = mul2(mul2(both(scale), w.p[j]), mul2(dz[i].p[j], ny[i].p[j]));
            if (f32) store8<kAccess>(row_of<float>(p.dgate, row), col, n, pack<float>(d));
            else store8<kAccess>(row_of<T>(p.dgate, row), col, n, pack<T>(d));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) dz[i].p[j] = mul2(dz[i].p[j], g.p[j]);
        }
        Vals sums_c;
        if constexpr (kLong) sums_c = accs.get8<float>(0, kAccC + i * 2);
        else sums_c = acc_c[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sums_c.p[j] = fma2(mul2(dz[i].p[j], both(row_gate)), ny[i].p[j], sums_c.p[j]);
          dz[i].p[j] = mul2(dz[i].p[j], w.p[j]);
          dot2 = fma2(dz[i].p[j], ny[i].p[j], dot2);
        }
        if constexpr (kLong) hold(accs, kAccC + i * 2, sums_c);
        else acc_c[i] = sums_c;
      }
      if constexpr (kForm == kRing) fetch(first + threadIdx.y + p.stages * step, stage);   // this thread has read its words
      const float dot = sum(sum2(dot2));
      if (live) acc_s = fmaf(row_gate, dot, acc_s);
      if (p.gate_kind == kRow && p.dgate.p && live && threadIdx.x == 0) {
        if (p.gate_f32) row_of<float>(p.dgate, row)[0] = scale * dot;
        else row_of<T>(p.dgate, row)[0] = from_float<T>(scale * dot);
      }
      if (wants_dy) {
        const float f = rstd1 * scale * row_gate, mean = dot * inv_n;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          Vals d;
#pragma unroll
          for (int j = 0; j < 4; ++j) d.p[j] = mul2(fma2(ny[i].p[j], both(-mean), dz[i].p[j]), both(f));
          store8<kAccess>(row_of<T>(p.dy, row), column(i), n, pack<T>(d));
        }
      }
    } else if constexpr (kForm == kRing) {
      fetch(first + threadIdx.y + p.stages * step, stage);
    }
    if constexpr (kForm == kRing)
      if (++stage == p.stages) stage = 0;
  }
  const long long group = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const long long at = group * ((p.n + 7) / 8 * 8);          // a group's sums are padded to whole eights
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    if constexpr (kMode != kPost) {
      if constexpr (kLong) acc_w2[0] = accs.get8<float>(0, i * 2);
      if (p.part_w2) store8<kAccess>(p.part_w2 + at, column(i), p.n, pack<float>(acc_w2[kLong ? 0 : i]));
    }
    if constexpr (kMode != kPre) {
      if constexpr (kLong) acc_c[0] = accs.get8<float>(0, kAccC + i * 2);
      if (p.part_c) store8<kAccess>(p.part_c + at, column(i), p.n, pack<float>(acc_c[kLong ? 0 : i]));
    }
  }
  if (kMode != kPre && p.part_s && threadIdx.x == 0) p.part_s[group] = acc_s;
}

// Threads of a row, rows of a block, eights of columns per thread and blocks for rows of n columns.
struct Shape { int threads, rows, chunks, blocks, form, stages, words, held; };
constexpr int kMaxColumns = 16384;
constexpr int kRingBytes = 216 * 1024;                // of a multiprocessor's shared memory, for all of its blocks

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

template <typename K, typename P> int launch(K* kernel, dim3 grid, dim3 block, int shared, const P& p, cudaStream_t stream) {
  if (shared > 40 * 1024)                             // 48 KB with the static part need no asking; the same for every call, or one of two at once lowered it
    BSHMEM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSHMEM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return 0;
}

// The ring of a block that shares its multiprocessor with `blocks - 1` others: as many stages as fit beside `held` words of weights,
// up to three (16384 x 4096 with a gate per element: 106 us with three, 108 with four, 109 with six).  Fewer than two: none.
inline void ring_of(Shape& s, int words, int held, int blocks) {
  s.words = words;
  s.held = held;
  s.stages = (kRingBytes / blocks / (16 * s.threads * s.rows) - held) / words;
  if (s.stages > 3) s.stages = 3;
}
inline int shared_of(const Shape& s) { return (s.stages * s.words + s.held) * 16 * s.threads * s.rows; }

// words(chunks): 16-byte words that a thread needs for one row.
template <typename F, typename G> Shape forward_shape(long long rows, int n, bool vec, int sms, F words, G ring_threads) {
  const int eights = (n + 7) / 8;
  Shape s = {};
  auto divide = [&](int chunks, int block) {
    s.chunks = chunks;
    s.threads = ((eights + chunks - 1) / chunks + 31) / 32 * 32;
    s.rows = s.threads >= block ? 1 : block / s.threads;
    if (s.rows > rows) s.rows = rows < 1 ? 1 : (int)rows;
  };
  if (vec) {
    // two eights a thread keep the weights in registers (4096 x 16384: 88 us for 153 with four); with 512 threads they end at 8192 columns
    divide(eights > 1024 && ring_threads(2) == 512 ? 4 : 2, 256);
    const int per_sm = ring_threads(s.chunks) / (s.threads * s.rows);
    const long long most = (long long)sms * per_sm;
    ring_of(s, words(s.chunks), 0, per_sm);
    if (s.stages >= 2 && rows > 2 * most * s.rows) {
      s.form = kRing;
      s.blocks = (int)most;
      return s;
    }
  }
  // few rows: as many threads for each as it has eights; many: four eights per thread, whose loads are all on their way at once
  divide(vec && rows <= 2LL * sms && eights <= 1024 ? 1 : 4, 128);
  s.form = vec ? kDirect : kScalar;
  s.blocks = (int)((rows + s.rows - 1) / s.rows);
  return s;
}
template <typename F, typename G> Shape backward_shape(long long rows, int n, bool vec, int sms, F words, G held, bool raw) {
  const int eights = (n + 7) / 8;
  Shape s = {};
  s.chunks = eights > 32 ? 2 : 1;
  s.threads = ((eights + s.chunks - 1) / s.chunks + 31) / 32 * 32;
  s.rows = s.threads >= 256 ? 1 : 256 / s.threads;
  if (s.rows > rows) s.rows = rows < 1 ? 1 : (int)rows;
  const long long need = (rows + s.rows - 1) / s.rows;
  const int per_sm = 512 / (s.threads * s.rows) < 1 ? 1 : 512 / (s.threads * s.rows);        // 128 registers a thread
  const long long most = (long long)sms * per_sm;
  s.blocks = (int)(need < most ? need : most);
  s.form = vec ? kDirect : kScalar;
  if (eights > 1024) {
    s.words = 0;
    s.held = held(s.chunks);                          // as many words as the weights: the column sums
  } else if (vec) {
    ring_of(s, words(s.chunks), held(s.chunks), per_sm);
    if (s.stages < 2 && raw) ring_of(s, words(s.chunks), held(s.chunks) / 2, per_sm);
    if (s.stages < 2) ring_of(s, words(s.chunks), 0, per_sm);
    if (s.stages >= 2 && need > most) s.form = kRing;
  }
  return s;
}

template <typename T, int kMode, bool kKeep, int kElement> int forward_ring(const Shape& s, const Params& p, dim3 grid, dim3 block, cudaStream_t stream) {
  if constexpr (ring_threads(kMode, 2, kKeep || kElement != kNone) == 512) {               // see forward_shape
    if (s.chunks == 4) return launch(norm_fwd_kernel<T, kMode, 4, kRing, kKeep, kElement>, grid, block, shared_of(s), p, stream);
  }
  return launch(norm_fwd_kernel<T, kMode, 2, kRing, kKeep, kElement>, grid, block, shared_of(s), p, stream);
}
template <typename T, int kMode, bool kKeep> int forward_ring(const Shape& s, const Params& p, dim3 grid, dim3 block, cudaStream_t stream) {
  if constexpr (kMode != kPre) {
    if (p.gate_kind == Gate::kElement) {
      if constexpr (sizeof(T) == 2) {
        if (p.gate_f32) return forward_ring<T, kMode, kKeep, kOfF32>(s, p, grid, block, stream);
      }
      return forward_ring<T, kMode, kKeep, kOfT>(s, p, grid, block, stream);
    }
  }
  return forward_ring<T, kMode, kKeep, kNone>(s, p, grid, block, stream);
}
template <typename T, int kMode> int forward_mode(bool vec, Params p, cudaStream_t stream) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int W = Raw8<T>::kWords, gate = p.gate_kind != kElement ? 0 : p.gate_f32 ? 2 : W;
  const Shape s = forward_shape(p.rows, p.n, vec, sms, [&](int chunks) { return chunks * (W * (kMode == kPre ? 1 : 2) + gate); },
                                [&](int chunks) { return ring_threads(kMode, chunks, p.q1 || p.q2 || gate); });
  const dim3 grid((unsigned)s.blocks), block(s.threads, s.rows);
  if (s.form == kRing) {
    p.stages = s.stages;
    p.ring_words = s.words;
    return p.q1 || p.q2 ? forward_ring<T, kMode, true>(s, p, grid, block, stream) : forward_ring<T, kMode, false>(s, p, grid, block, stream);
  }
  if (s.form == kScalar) return launch(norm_fwd_kernel<T, kMode, 4, kScalar>, grid, block, 0, p, stream);
  if (s.chunks == 1) return launch(norm_fwd_kernel<T, kMode, 1, kDirect>, grid, block, 0, p, stream);
  return launch(norm_fwd_kernel<T, kMode, 4, kDirect>, grid, block, 0, p, stream);
}
// The words of norm_bwd_kernel's stages.
inline int backward_words(int size, int mode, bool kept, int gate_kind, bool gate_f32, int chunks) {
  const int W = size / 2, K = kept ? 1 : W;
  return chunks * ((mode == kPostPre ? 2 : 1) * (W + K) + (gate_kind != kElement ? 0 : gate_f32 ? 2 : W)) + 1;
}
inline int backward_held(int mode, int chunks) { return chunks * 2 * (mode == kPostPre ? 2 : 1); }
// Whether half of that will do: 2-byte rows, weights of their type or none, no gate per column, which is multiplied into w1.
inline bool backward_raw(const BwdParams& p, int size) {
  return size == 2 && p.gate_kind != kColumn && !(p.w1 && p.w1_f32) && !(p.w2 && p.w2_f32);
}
template <typename T, int kMode, bool kKept, int kHeld> int backward_usual(dim3 grid, dim3 block, int shared, const BwdParams& p, cudaStream_t stream) {
  if constexpr (kMode != kPre) {
    if (p.gate_kind == Gate::kElement) {
      if (sizeof(T) == 2 && p.gate_f32) return launch(norm_bwd_kernel<T, kMode, 2, kRing, kKept>, grid, block, shared, p, stream);
      return launch(norm_bwd_kernel<T, kMode, 2, kRing, kKept, kHeld, kOfT>, grid, block, shared, p, stream);
    }
  }
  return launch(norm_bwd_kernel<T, kMode, 2, kRing, kKept, kHeld, kNone>, grid, block, shared, p, stream);
}
template <typename T, int kMode, bool kKept> int backward_mode(const Shape& s, BwdParams p, cudaStream_t stream) {
  const dim3 grid((unsigned)s.blocks), block(s.threads, s.rows);
  if (s.threads > 512) {
    if (s.form == kDirect) return launch(norm_bwd_kernel<T, kMode, 2, kDirect, kKept, 0, kAsk, true>, grid, block, shared_of(s), p, stream);
    return launch(norm_bwd_kernel<T, kMode, 2, kScalar, kKept, 0, kAsk, true>, grid, block, shared_of(s), p, stream);
  }
  if (s.form == kRing) {
    p.stages = s.stages;
    p.ring_words = s.words;
    p.held = s.held == 0 ? 0 : s.held == backward_held(kMode, s.chunks) ? 1 : 2;
    const int shared = shared_of(s);
    if (s.chunks == 1) return launch(norm_bwd_kernel<T, kMode, 1, kRing, kKept>, grid, block, shared, p, stream);
    if (p.held == 0 || (kMode != kPre && !(p.dout.p && p.dy.p))) return launch(norm_bwd_kernel<T, kMode, 2, kRing, kKept>, grid, block, shared, p, stream);
    if constexpr (sizeof(T) == 2) {
      if (p.held == 2) return backward_usual<T, kMode, kKept, 2>(grid, block, shared, p, stream);
    }
    return backward_usual<T, kMode, kKept, 1>(grid, block, shared, p, stream);
  }
  if (s.form == kDirect) {
    if (s.chunks == 1) return launch(norm_bwd_kernel<T, kMode, 1, kDirect, kKept>, grid, block, 0, p, stream);
    return launch(norm_bwd_kernel<T, kMode, 2, kDirect, kKept>, grid, block, 0, p, stream);
  }
  if (s.chunks == 1) return launch(norm_bwd_kernel<T, kMode, 1, kScalar, kKept>, grid, block, 0, p, stream);
  return launch(norm_bwd_kernel<T, kMode, 2, kScalar, kKept>, grid, block, 0, p, stream);
}

// The kernels for one type of rows; norm_bf16.cu, norm_fp16.cu and norm_fp32.cu instantiate them.
template <typename T> int forward(int mode, bool vec, const Params& p, cudaStream_t stream) {
  return mode == kPre ? forward_mode<T, kPre>(vec, p, stream) : mode == kPost ? forward_mode<T, kPost>(vec, p, stream)
                                                                              : forward_mode<T, kPostPre>(vec, p, stream);
}
template <typename T> int backward(int mode, bool kept, const Shape& s, const BwdParams& p, cudaStream_t stream) {
  if (mode == kPre) return kept ? backward_mode<T, kPre, true>(s, p, stream) : backward_mode<T, kPre, false>(s, p, stream);
  if (mode == kPost) return kept ? backward_mode<T, kPost, true>(s, p, stream) : backward_mode<T, kPost, false>(s, p, stream);
  return kept ? backward_mode<T, kPostPre, true>(s, p, stream) : backward_mode<T, kPostPre, false>(s, p, stream);
}

}  // namespace norms
}  // namespace bshmem
