// checkpoint8.cu — activations in 8 bits between the forward and the backward pass (the form is in row_values.cuh): to it and
// back, and the gated activation act = silu(gate) * up that keeps its input so.
//
// Every kernel reads and writes each byte once and computes next to nothing: memory bounds them.  A thread has eight columns and
// sixteen threads a block of 128, so the largest value of a block is found by four shuffles.
#include "ptx.cuh"
#include "row_values.cuh"
#include "tma_host.h"

using namespace bshmem;
using namespace bshmem::rows;

namespace {

constexpr int kThreads = 256;

struct StoreParams { const void* x; long long ldx; uint8_t* q; uint8_t* e; long long ldq, lde, rows; int n; long long eights; };

// Thread i of the grid has the i-th eight of its row; rows are padded to whole blocks of 128 columns (16 threads).
template <typename T, int kAccess> __global__ void __launch_bounds__(kThreads) store8_kernel(const StoreParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i / p.eights;
  const int col = (int)(i - row * p.eights) * 8;
  const int n = row < p.rows ? p.n : 0;
  const Vals v = unpack(load8<kAccess>(static_cast<const T*>(p.x) + (n ? row * p.ldx : 0), col, n));
  uint32_t e;
  const uint2 q = encode8<T>(v, e);
  if (col < n) {
    *reinterpret_cast<uint2*>(p.q + row * p.ldq + col) = q;
    if (col % 128 == 0) p.e[row * p.lde + col / 128] = (uint8_t)e;
  }
}

struct RestoreParams { const uint8_t *q, *e; long long ldq, lde; void* x; long long ldx, rows; int n; long long eights; };

template <typename T, int kAccess> __global__ void __launch_bounds__(kThreads) restore8_kernel(const RestoreParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i / p.eights;
  if (row >= p.rows) return;
  const int col = (int)(i - row * p.eights) * 8;
  if (col >= p.n) return;
  const Vals v = decode8(__ldg(reinterpret_cast<const uint2*>(p.q + row * p.ldq + col)), __ldg(p.e + row * p.lde + col / 128));
  store8<kAccess>(static_cast<T*>(p.x) + row * p.ldx, col, p.n, pack<T>(v));
}

// gu: [rows, 2F], 32 columns of the gate and the 32 of `up` that belong to them in turn.
struct SwigluParams {
  const __nv_bfloat16 *gu, *dact;
  __nv_bfloat16 *act, *dgu;
  uint8_t *q, *e;
  long long lde, rows;
  int F;
  long long eights;                                   // of a row of gu, in whole blocks of 128 columns
};

__device__ __forceinline__ float2 sigmoid2(float2 x) { return make_float2(1.f / (1.f + __expf(-x.x)), 1.f / (1.f + __expf(-x.y))); }

// Thread i has eight columns of gu; four threads in a row have a gate, the next four its `up`, which they swap.
__global__ void __launch_bounds__(kThreads) swiglu_store8_kernel(const SwigluParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i / p.eights;
  const int col = (int)(i - row * p.eights) * 8;
  const int n = row < p.rows ? 2 * p.F : 0;
  const Raw8<__nv_bfloat16> r = load8<kVector>(p.gu + (n ? row * n : 0), col, n);
  const Vals v = unpack(r);
  uint32_t e;
  const uint2 q = encode8<__nv_bfloat16>(v, e);
  const uint4 w = r.get(0);
  Raw8<__nv_bfloat16> other;
  other.set(0, make_uint4(__shfl_xor_sync(0xffffffffu, w.x, 4), __shfl_xor_sync(0xffffffffu, w.y, 4), __shfl_xor_sync(0xffffffffu, w.z, 4),
                          __shfl_xor_sync(0xffffffffu, w.w, 4)));
  if (col >= n) return;
  *reinterpret_cast<uint2*>(p.q + row * n + col) = q;
  if (col % 128 == 0) p.e[row * p.lde + col / 128] = (uint8_t)e;
  if (col & 32) return;
  Vals u = unpack(other);
#pragma unroll
  for (int j = 0; j < 4; ++j) u.p[j] = mul2(u.p[j], mul2(v.p[j], sigmoid2(v.p[j])));
  store8<kVector>(p.act + row * p.F, col / 64 * 32 + col % 32, p.F, pack<__nv_bfloat16>(u));
}

// Thread i has eight columns of the activation: their gate and `up` in 8 bits lie 32 columns apart in one block.
template <bool kAct> __global__ void __launch_bounds__(kThreads) swiglu_backward8_kernel(const SwigluParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i / p.eights;
  if (row >= p.rows) return;
  const int col = (int)(i - row * p.eights) * 8;
  if (col >= p.F) return;
  const int at = col / 32 * 64 + col % 32;
  const uint8_t* q = p.q + row * 2 * p.F + at;
  const uint32_t e = __ldg(p.e + row * p.lde + at / 128);
  const Vals g = decode8(__ldg(reinterpret_cast<const uint2*>(q)), e), u = decode8(__ldg(reinterpret_cast<const uint2*>(q + 32)), e);
  const Vals d = unpack(load8<kVector>(p.dact + row * p.F, col, p.F));
  Vals dg, du, again;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 s = sigmoid2(g.p[j]), silu = mul2(g.p[j], s);
    du.p[j] = mul2(d.p[j], silu);
    again.p[j] = mul2(u.p[j], silu);
    // s (1 + g (1 - s)) = s + silu (1 - s)
    dg.p[j] = mul2(mul2(d.p[j], u.p[j]), fma2(silu, make_float2(1.f - s.x, 1.f - s.y), s));
  }
  __nv_bfloat16* o = p.dgu + row * 2 * p.F + at;
  store8<kVector>(o, 0, 8, pack<__nv_bfloat16>(dg));
  store8<kVector>(o, 32, 40, pack<__nv_bfloat16>(du));
  if constexpr (kAct) store8<kVector>(p.act + row * p.F, col, p.F, pack<__nv_bfloat16>(again));
}

template <typename K, typename P> int launch(K* kernel, long long threads, const P& p, void* stream) {
  const long long blocks = (threads + kThreads - 1) / kThreads;
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
// columns].  Bytes of q behind the last eight columns are not written.
int bshmem_ckpt8_store(int type, const void* x, long long ldx, void* kept, long long rows, int n, void* stream) {
  if (type < 0 || type > 2 || n < 1) { host::last_error() = "checkpoint: unknown type or no columns"; return 1; }
  if (rows <= 0) return 0;
  const long long blocks = ((long long)n + 127) / 128;
  const long long ldq = ((long long)n + 15) / 16 * 16;
  uint8_t* const q = static_cast<uint8_t*>(kept);
  const StoreParams p = {x, ldx, q, q + rows * ldq, ldq, blocks, rows, n, blocks * 16};
  const bool vec = n % 8 == 0 && aligned(x) && ldx * (type == 2 ? 4 : 2) % 16 == 0;
  const long long threads = rows * p.eights;
  if (type == 0) return vec ? launch(store8_kernel<__nv_bfloat16, kVector>, threads, p, stream) : launch(store8_kernel<__nv_bfloat16, kSingle>, threads, p, stream);
  if (type == 1) return vec ? launch(store8_kernel<__half, kVector>, threads, p, stream) : launch(store8_kernel<__half, kSingle>, threads, p, stream);
  return vec ? launch(store8_kernel<float, kVector>, threads, p, stream) : launch(store8_kernel<float, kSingle>, threads, p, stream);
}

// The way back; x has row pitch ldx.
int bshmem_ckpt8_restore(int type, const void* kept, void* x, long long ldx, long long rows, int n, void* stream) {
  if (type < 0 || type > 2 || n < 1) { host::last_error() = "checkpoint: unknown type or no columns"; return 1; }
  if (rows <= 0) return 0;
  const long long ldq = ((long long)n + 15) / 16 * 16;
  const uint8_t* const q = static_cast<const uint8_t*>(kept);
  const RestoreParams p = {q, q + rows * ldq, ldq, ((long long)n + 127) / 128, x, ldx, rows, n, ((long long)n + 7) / 8};
  const bool vec = n % 8 == 0 && aligned(x) && ldx * (type == 2 ? 4 : 2) % 16 == 0;
  const long long threads = rows * p.eights;
  if (type == 0) return vec ? launch(restore8_kernel<__nv_bfloat16, kVector>, threads, p, stream) : launch(restore8_kernel<__nv_bfloat16, kSingle>, threads, p, stream);
  if (type == 1) return vec ? launch(restore8_kernel<__half, kVector>, threads, p, stream) : launch(restore8_kernel<__half, kSingle>, threads, p, stream);
  return vec ? launch(restore8_kernel<float, kVector>, threads, p, stream) : launch(restore8_kernel<float, kSingle>, threads, p, stream);
}

// gu [rows, 2F] bf16 -> act [rows, F] and gu in 8 bits.  Everything contiguous and 16-byte aligned, F % 32 == 0.
int bshmem_ckpt8_swiglu_store(const void* gu, void* act, void* kept, long long rows, int F, void* stream) {
  if (F < 32 || F % 32 || F > 1 << 29 || !aligned(gu) || !aligned(act)) { host::last_error() = "checkpoint: swiglu needs F % 32 == 0 and 16-byte aligned rows"; return 1; }
  if (rows <= 0) return 0;
  SwigluParams p = {};
  p.gu = static_cast<const __nv_bfloat16*>(gu);
  p.act = static_cast<__nv_bfloat16*>(act);
  p.q = static_cast<uint8_t*>(kept); p.e = p.q + rows * 2 * F;
  p.lde = (2LL * F + 127) / 128; p.rows = rows; p.F = F; p.eights = p.lde * 16;
  return launch(swiglu_store8_kernel, rows * p.eights, p, stream);
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
  p.lde = (2LL * F + 127) / 128; p.rows = rows; p.F = F; p.eights = F / 8;
  return act ? launch(swiglu_backward8_kernel<true>, rows * p.eights, p, stream) : launch(swiglu_backward8_kernel<false>, rows * p.eights, p, stream);
}

}  // extern "C"
