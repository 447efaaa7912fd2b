// checkpoint8.cu — activations in 8 bits between the forward and the backward pass (the form is in row_values.cuh): to it and
// back, and the gated activation act = silu(gate) * up that keeps its input so.
//
// Every kernel reads and writes each byte once: memory bounds them, but for the way to the form, where conversions come close to what the
// multiprocessors issue.  8192 x 3584 of the gated activation, forward and backward: 84 us (6.3 TB/s).
#include "ptx.cuh"
#include "row_values.cuh"
#include "tma_host.h"

using namespace bshmem;
using namespace bshmem::rows;

namespace {

constexpr int kThreads = 256;

// A thread has several eights, whose loads are all on their way before the first is used: with one alone, 32 KB of an SM on their way,
// 16384 x 4096 there and back took 83 us, for 76 with four.  On the way there two of them are of one block of 128 columns, whose largest value
// takes eight threads then: it is bound by issue (three instructions a cycle with one eight of a block for each of sixteen threads), and there and
// back take 70 us so, 67 with plain loads (6.1 TB/s).
constexpr int kPer = 4, kPairs = 2;
struct Eights { long long total; uint32_t per_row; };
// Row and column of the i-th eight; a 64-bit division only where there are that many.
__device__ __forceinline__ void place(const Eights& s, long long i, long long& row, int& col) {
  uint32_t in;
  if (s.total <= 0xffffffffLL) {
    const uint32_t r = (uint32_t)i / s.per_row;
    in = (uint32_t)i - r * s.per_row;
    row = r;
  } else {
    row = i / s.per_row;
    in = (uint32_t)(i - row * s.per_row);
  }
  col = (int)in * 8;
}

struct StoreParams { const void* x; long long ldx; uint8_t* q; uint8_t* e; long long ldq, lde; int n; Eights size; };

// The size counts pairs of eights: the j-th and the (j + 8)-th of a block are thread j's.
template <typename T, int kAccess> __global__ void __launch_bounds__(kThreads) store8_kernel(const StoreParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPairs) + threadIdx.x;
  long long row[kPairs];
  int col[kPairs], n[kPairs];
  Raw8<T> r[kPairs][2];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const long long i = first + j * kThreads;
    n[j] = i < p.size.total ? p.n : 0;
    place(p.size, n[j] ? i : 0, row[j], col[j]);
    col[j] = col[j] / 64 * 128 + col[j] % 64;
#pragma unroll
    for (int k = 0; k < 2; ++k) r[j][k] = load8<kAccess>(static_cast<const T*>(p.x) + row[j] * p.ldx, col[j] + 64 * k, n[j]);
  }
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    uint32_t e;
    uint2 q[2];
    encode<T, 2>({unpack(r[j][0]), unpack(r[j][1])}, q, e);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (col[j] + 64 * k < byte_columns(n[j])) *reinterpret_cast<uint2*>(p.q + row[j] * p.ldq + col[j] + 64 * k) = q[k];
    if (col[j] % 128 == 0 && col[j] < n[j]) p.e[row[j] * p.lde + col[j] / 128] = (uint8_t)e;
  }
}

struct RestoreParams { const uint8_t *q, *e; long long ldq, lde; void* x; long long ldx; int n; Eights size; };

template <typename T, int kAccess> __global__ void __launch_bounds__(kThreads) restore8_kernel(const RestoreParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPer) + threadIdx.x;
  long long row[kPer];
  int col[kPer];
  uint2 q[kPer];
  uint32_t e[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    place(p.size, min(first + j * kThreads, p.size.total - 1), row[j], col[j]);
    q[j] = *reinterpret_cast<const uint2*>(p.q + row[j] * p.ldq + col[j]);
    e[j] = p.e[row[j] * p.lde + col[j] / 128];
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (first + j * kThreads < p.size.total) store8<kAccess>(static_cast<T*>(p.x) + row[j] * p.ldx, col[j], p.n, pack<T>(decode8(q[j], e[j])));
}

// gu: [rows, 2F], 32 columns of the gate and the 32 of `up` that belong to them in turn.
struct SwigluParams {
  const __nv_bfloat16 *gu, *dact;
  __nv_bfloat16 *act, *dgu;
  uint8_t *q, *e;
  long long lde;
  int F;
  Eights size;                                        // of the activation; forward: in whole blocks
};

__device__ __forceinline__ float2 sigmoid2(float2 x) { return make_float2(1.f / (1.f + __expf(-x.x)), 1.f / (1.f + __expf(-x.y))); }

// A thread has eights of the activation; the gate and `up` of eight threads are a block.  Without kKeep only the activation is written.
template <bool kKeep> __global__ void __launch_bounds__(kThreads) swiglu_store8_kernel(const SwigluParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPairs) + threadIdx.x;
  long long row[kPairs];
  int col[kPairs], at[kPairs];
  bool in[kPairs];
  Raw8<__nv_bfloat16> r[kPairs][2];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const long long i = first + j * kThreads;
    place(p.size, i < p.size.total ? i : 0, row[j], col[j]);
    in[j] = i < p.size.total && col[j] < p.F;
    at[j] = col[j] / 32 * 64 + col[j] % 32;
#pragma unroll
    for (int k = 0; k < 2; ++k) r[j][k] = load8<kVector>(p.gu + row[j] * 2 * p.F, at[j] + 32 * k, in[j] ? 2 * p.F : 0);
  }
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const Vals g = unpack(r[j][0]), u = unpack(r[j][1]);
    if constexpr (kKeep) {
      uint32_t e;
      uint2 q[2];
      encode<__nv_bfloat16, 2>({g, u}, q, e);
      if (in[j]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) *reinterpret_cast<uint2*>(p.q + row[j] * 2 * p.F + at[j] + 32 * k) = q[k];
        if (at[j] % 128 == 0) p.e[row[j] * p.lde + at[j] / 128] = (uint8_t)e;
      }
    }
    Vals o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o.p[k] = mul2(u.p[k], mul2(g.p[k], sigmoid2(g.p[k])));
    if (in[j]) store8<kVector>(p.act + row[j] * p.F, col[j], p.F, pack<__nv_bfloat16>(o));
  }
}

// A thread has eights of the activation, whose gate and `up` lie 32 bytes apart in one block.
constexpr int kPerBack = 2;
template <bool kAct> __global__ void __launch_bounds__(kThreads) swiglu_backward8_kernel(const SwigluParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPerBack) + threadIdx.x;
  long long row[kPerBack];
  int col[kPerBack], at[kPerBack];
  uint2 qg[kPerBack], qu[kPerBack];
  uint32_t e[kPerBack];
  Raw8<__nv_bfloat16> rd[kPerBack];
#pragma unroll
  for (int j = 0; j < kPerBack; ++j) {
    place(p.size, min(first + j * kThreads, p.size.total - 1), row[j], col[j]);
    at[j] = col[j] / 32 * 64 + col[j] % 32;
    const uint8_t* q = p.q + row[j] * 2 * p.F + at[j];
    e[j] = p.e[row[j] * p.lde + at[j] / 128];
    qg[j] = *reinterpret_cast<const uint2*>(q);
    qu[j] = *reinterpret_cast<const uint2*>(q + 32);
    rd[j] = load8<kVector>(p.dact + row[j] * p.F, col[j], p.F);
  }
#pragma unroll
  for (int j = 0; j < kPerBack; ++j) {
    if (first + j * kThreads >= p.size.total) continue;
    const Vals g = decode8(qg[j], e[j]), u = decode8(qu[j], e[j]), d = unpack(rd[j]);
    Vals dg, du, again;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 s = sigmoid2(g.p[k]), silu = mul2(g.p[k], s);
      du.p[k] = mul2(d.p[k], silu);
      again.p[k] = mul2(u.p[k], silu);
      // s (1 + g (1 - s)) = s + silu (1 - s)
      dg.p[k] = mul2(mul2(d.p[k], u.p[k]), fma2(silu, make_float2(1.f - s.x, 1.f - s.y), s));
    }
    __nv_bfloat16* o = p.dgu + row[j] * 2 * p.F + at[j];
    store8<kVector>(o, 0, 8, pack<__nv_bfloat16>(dg));
    store8<kVector>(o, 32, 40, pack<__nv_bfloat16>(du));
    if constexpr (kAct) store8<kVector>(p.act + row[j] * p.F, col[j], p.F, pack<__nv_bfloat16>(again));
  }
}

template <typename K, typename P> int launch(K* kernel, int per, const P& p, void* stream) {
  const long long blocks = (p.size.total + kThreads * per - 1) / (kThreads * per);
  if (blocks > 0x7fffffffLL) { host::last_error() = "checkpoint: too many elements for one call"; return 1; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSHMEM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return 0;
}

bool aligned(const void* p) { return !(reinterpret_cast<uintptr_t>(p) & 15); }

}  // namespace

extern "C" {

const char* bshmem_ckpt8_last_error() { return host::last_error().c_str(); }

// x: [rows, n] of type 0 bf16, 1 fp16, 2 fp32 with row pitch ldx -> kept: q [rows][n rounded up to 16], then e [rows][blocks of 128
// columns].  The columns that q has beyond n are zeros.
int bshmem_ckpt8_store(int type, const void* x, long long ldx, void* kept, long long rows, int n, void* stream) {
  if (type < 0 || type > 2 || n < 1) { host::last_error() = "checkpoint: unknown type or no columns"; return 1; }
  if (rows <= 0) return 0;
  const long long blocks = ((long long)n + 127) / 128;
  const long long ldq = ((long long)n + 15) / 16 * 16;
  uint8_t* const q = static_cast<uint8_t*>(kept);
  const StoreParams p = {x, ldx, q, q + rows * ldq, ldq, blocks, n, {rows * blocks * 8, (uint32_t)(blocks * 8)}};
  const bool vec = n % 8 == 0 && aligned(x) && ldx * (type == 2 ? 4 : 2) % 16 == 0;
  if (type == 0) return vec ? launch(store8_kernel<__nv_bfloat16, kVector>, kPairs, p, stream) : launch(store8_kernel<__nv_bfloat16, kSingle>, kPairs, p, stream);
  if (type == 1) return vec ? launch(store8_kernel<__half, kVector>, kPairs, p, stream) : launch(store8_kernel<__half, kSingle>, kPairs, p, stream);
  return vec ? launch(store8_kernel<float, kVector>, kPairs, p, stream) : launch(store8_kernel<float, kSingle>, kPairs, p, stream);
}

// The way back; x has row pitch ldx.
int bshmem_ckpt8_restore(int type, const void* kept, void* x, long long ldx, long long rows, int n, void* stream) {
  if (type < 0 || type > 2 || n < 1) { host::last_error() = "checkpoint: unknown type or no columns"; return 1; }
  if (rows <= 0) return 0;
  const long long ldq = ((long long)n + 15) / 16 * 16;
  const uint8_t* const q = static_cast<const uint8_t*>(kept);
  const RestoreParams p = {q, q + rows * ldq, ldq, ((long long)n + 127) / 128, x, ldx, n,
                           {rows * (((long long)n + 7) / 8), (uint32_t)(((long long)n + 7) / 8)}};
  const bool vec = n % 8 == 0 && aligned(x) && ldx * (type == 2 ? 4 : 2) % 16 == 0;
  if (type == 0) return vec ? launch(restore8_kernel<__nv_bfloat16, kVector>, kPer, p, stream) : launch(restore8_kernel<__nv_bfloat16, kSingle>, kPer, p, stream);
  if (type == 1) return vec ? launch(restore8_kernel<__half, kVector>, kPer, p, stream) : launch(restore8_kernel<__half, kSingle>, kPer, p, stream);
  return vec ? launch(restore8_kernel<float, kVector>, kPer, p, stream) : launch(restore8_kernel<float, kSingle>, kPer, p, stream);
}

// gu [rows, 2F] bf16 -> act [rows, F] and, unless kept is null, gu in 8 bits.  Everything contiguous and 16-byte aligned, F % 32 == 0.
int bshmem_ckpt8_swiglu_store(const void* gu, void* act, void* kept, long long rows, int F, void* stream) {
  if (F < 32 || F % 32 || F > 1 << 29 || !aligned(gu) || !aligned(act)) { host::last_error() = "checkpoint: swiglu needs F % 32 == 0 and 16-byte aligned rows"; return 1; }
  if (rows <= 0) return 0;
  SwigluParams p = {};
  p.gu = static_cast<const __nv_bfloat16*>(gu);
  p.act = static_cast<__nv_bfloat16*>(act);
  p.q = static_cast<uint8_t*>(kept); p.e = p.q + rows * 2 * F;
  p.lde = (2LL * F + 127) / 128; p.F = F;
  p.size = {rows * p.lde * 8, (uint32_t)(p.lde * 8)};
  return kept ? launch(swiglu_store8_kernel<true>, kPairs, p, stream) : launch(swiglu_store8_kernel<false>, kPairs, p, stream);
}

// dgu [rows, 2F] from gu in 8 bits and dact [rows, F]; act (may be null): the activation again, of the same 8 bits.
int bshmem_ckpt8_swiglu_backward(const void* kept, const void* dact, void* dgu, void* act, long long rows, int F, void* stream) {
  if (F < 32 || F % 32 || F > 1 << 29 || !aligned(dact) || !aligned(dgu) || !aligned(act)) { host::last_error() = "checkpoint: swiglu needs F % 32 == 0 and 16-byte aligned rows"; return 1; }
  if (rows <= 0) return 0;
  SwigluParams p = {};
  p.q = static_cast<uint8_t*>(const_cast<void*>(kept)); p.e = p.q + rows * 2 * F;
  p.dact = static_cast<const __nv_bfloat16*>(dact);
  p.dgu = static_cast<__nv_bfloat16*>(dgu);
  p.act = static_cast<__nv_bfloat16*>(act);
  p.lde = (2LL * F + 127) / 128; p.F = F;
  p.size = {rows * (F / 8), (uint32_t)(F / 8)};
  return act ? launch(swiglu_backward8_kernel<true>, kPerBack, p, stream) : launch(swiglu_backward8_kernel<false>, kPerBack, p, stream);
}

}  // extern "C"
