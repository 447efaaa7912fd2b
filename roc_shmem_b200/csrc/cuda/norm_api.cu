// norm_api.cu — C entry points of the norms: argument checks, the choice of a kernel, and the sums over the groups of rows that
// end a backward pass.
#include <cstring>

#include "norm_kernels.cuh"

using namespace bshmem;
using namespace bshmem::norms;

namespace bshmem {
namespace norms {
extern template int forward<__nv_bfloat16>(int, bool, const Params&, cudaStream_t);
extern template int forward<__half>(int, bool, const Params&, cudaStream_t);
extern template int forward<float>(int, bool, const Params&, cudaStream_t);
extern template int backward<__nv_bfloat16>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
extern template int backward<__half>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
extern template int backward<float>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
}  // namespace norms
}  // namespace bshmem

namespace {

struct FinishParams {
  const float *part_w2, *part_c, *part_s;
  const void *w1, *gcol, *scale;
  float scale_value;
  void *dw1, *dw2, *dgcol, *dscale;
  long long groups;
  int n;
  int w1_f32, w2_f32, gcol_f32, scale_f32;            // fp32, or the rows' type
};

template <typename T> __device__ __forceinline__ void put(void* p, int f32, long long i, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = rows::from_float<T>(v);
}
template <typename T> __device__ __forceinline__ float at(const void* p, int f32, long long i) {
  return !p ? 1.f : f32 ? static_cast<const float*>(p)[i] : rows::to_float<T>(static_cast<const T*>(p)[i]);
}

constexpr int kFinishCols = 32, kFinishLanes = 32;    // columns and lanes of groups of a block

// Column sums of the groups: lane (x, y) adds up groups y, y + 32, ... of its column, four on their way at a time, then the 32 sums are
// added in their order.  What counts is how many loads are on their way: one load after the other took 13.5 us for 296
// groups of 4096 columns.
template <typename T> __global__ void __launch_bounds__(kFinishCols * kFinishLanes) norm_bwd_finish_kernel(const FinishParams p) {
  __shared__ float tile[2][kFinishLanes][kFinishCols + 1];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int col = blockIdx.x * kFinishCols + threadIdx.x;
  const long long pitch = (p.n + 7) / 8 * 8;
  float a = 0.f, c = 0.f;
  if (col < p.n)
    for (long long g = threadIdx.y; g < p.groups; g += 4 * kFinishLanes) {
      float va[4], vc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long at = g + i * kFinishLanes;
        va[i] = p.part_w2 && at < p.groups ? p.part_w2[at * pitch + col] : 0.f;
        vc[i] = p.part_c && at < p.groups ? p.part_c[at * pitch + col] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { a += va[i]; c += vc[i]; }
    }
  tile[0][threadIdx.y][threadIdx.x] = a;
  tile[1][threadIdx.y][threadIdx.x] = c;
  __syncthreads();
  const float scale = number<T>(p.scale, p.scale_f32, p.scale_value);
  if (threadIdx.y < 2 && col < p.n) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kFinishLanes; ++i) s += tile[threadIdx.y][i][threadIdx.x];
    if (threadIdx.y == 0) {
      if (p.dw2) put<T>(p.dw2, p.w2_f32, col, s);
    } else {
      if (p.dw1) put<T>(p.dw1, p.w1_f32, col, scale * s * at<T>(p.gcol, p.gcol_f32, col));
      if (p.dgcol) put<T>(p.dgcol, p.gcol_f32, col, scale * s * at<T>(p.w1, p.w1_f32, col));
    }
  }
  if (blockIdx.x == 0 && p.dscale) {
    __syncthreads();
    constexpr int kThreads = kFinishCols * kFinishLanes, kWarps = kThreads / 32;
    float s = 0.f;
    const int t = threadIdx.y * kFinishCols + threadIdx.x;
    for (long long g = t; g < p.groups; g += kThreads) s += p.part_s[g];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (t % 32 == 0) tile[0][t / 32][0] = s;
    __syncthreads();
    if (t == 0) {
      s = 0.f;
      for (int i = 0; i < kWarps; ++i) s += tile[0][i][0];
      put<T>(p.dscale, p.scale_f32, 0, s);
    }
  }
}

bool aligned(const void* p) { return !(reinterpret_cast<uintptr_t>(p) & 15); }
bool aligned(const Mat& m, int size) { return aligned(m.p) && (m.ld * size) % 16 == 0; }

// The number of groups goes by the sizes alone (see backward_shape): the rows' layout chooses between forms of the same shape.
int groups_of(long long rows, int n, int* groups) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const Shape s = backward_shape(rows, n, false, sms, [](int) { return 1; }, [](int) { return 0; }, false);
  *groups = s.blocks * s.rows;
  return 0;
}

}  // namespace

extern "C" {

const char* bshmem_norm_last_error() { return host::last_error().c_str(); }

// Number of groups of rows whose column sums a backward pass leaves: part_w2 and part_c are [groups][n rounded up to 8] floats,
// part_s [groups].  Negative: an error.
int bshmem_norm_bwd_groups(long long rows, int n) {
  int groups = 0;
  if (rows < 1 || n < 1 || n > kMaxColumns) { host::last_error() = "norm: needs at least one row and 1 to 16384 columns"; return -1; }
  if (groups_of(rows, n, &groups)) return -7;
  return groups;
}

// What a call is, in one word: bits 0-1 type of the rows (0 bf16, 1 fp16, 2 fp32), 2-3 mode, 4-5 gate, and which operands are
// fp32 rather than of the rows' type: 8 w1, 9 w2, 10 gate, 11 scale; 12: y and z are kept in 8 bits.
struct Call {
  int type, mode, gate, w1_f32, w2_f32, gate_f32, scale_f32, kept, size;
  explicit Call(int f)
      : type(f & 3), mode(f >> 2 & 3), gate(f >> 4 & 3), w1_f32(f >> 8 & 1), w2_f32(f >> 9 & 1), gate_f32(f >> 10 & 1),
        scale_f32(f >> 11 & 1), kept(f >> 12 & 1), size((f & 3) == 2 ? 4 : 2) {}
  bool known() const { return type <= 2 && mode <= 2; }
};

static float float_of(uint64_t bits) {
  const uint32_t b = (uint32_t)bits;
  float f;
  memcpy(&f, &b, 4);
  return f;
}
static int refuse_size() {
  host::last_error() = "norm: unknown type or mode, or not 1 to 16384 columns and less than 2^31 rows";
  return 1;
}

// out and h are contiguous; rstd: [rows], in kPostPre [2][rows] (y's, then out's), or null.  kept: q [norms][rows][n rounded up to 16],
// then e [norms][rows][blocks of 128 columns], in the same order, 16-byte aligned and in whole 4-byte words; what has no value is zero.  numbers: the bits of eps,
// and of a scale that is not in memory above them.
int bshmem_norm_fwd(int what, const void* y, long long ldy, const void* x, long long ldx, void* out, void* h, const void* w1,
                    const void* w2, const void* gate, long long ldg, const void* scale, uint64_t numbers, void* rstd, void* kept,
                    long long rows, int n, void* stream) {
  const Call c(what);
  if (!c.known() || n < 1 || n > kMaxColumns || rows > 0x7fffffffLL) return refuse_size();
  if (rows <= 0) return 0;
  Params p = {};
  p.y = {const_cast<void*>(y), ldy};
  p.x = {const_cast<void*>(x), ldx};
  p.out = {out, n};
  p.h = {h, n};
  p.w1 = w1; p.w2 = w2;
  p.gate_kind = c.gate;
  if (c.gate == kColumn) p.gcol = gate;
  else p.gate = {const_cast<void*>(gate), ldg};
  p.gcol_f32 = p.gate_f32 = c.gate_f32;
  p.scale = scale; p.scale_f32 = c.scale_f32; p.scale_value = float_of(numbers >> 32);
  p.eps = float_of(numbers);
  p.w1_f32 = c.w1_f32; p.w2_f32 = c.w2_f32;
  p.rows = rows; p.n = n;
  if (rstd) {
    float* r = static_cast<float*>(rstd);
    p.rstd1 = c.mode == kPre ? nullptr : r;
    p.rstd2 = c.mode == kPost ? nullptr : c.mode == kPre ? r : r + rows;
  }
  if (c.kept) {
    p.ldq = (n + 15) / 16 * 16;
    p.lde = (n + 127) / 128;
    uint8_t *qb = static_cast<uint8_t*>(kept), *eb = qb + (c.mode == kPostPre ? 2 : 1) * rows * p.ldq;
    const long long exponents = (c.mode == kPostPre ? 2 : 1) * rows * p.lde;
    p.end = eb + exponents;
    p.tail = (int)(-exponents & 3);                     // q is whole words
    if (c.mode != kPre) { p.q1 = qb; p.e1 = eb; }
    if (c.mode != kPost) { p.q2 = qb + (c.mode == kPre ? 0 : rows * p.ldq); p.e2 = eb + (c.mode == kPre ? 0 : rows * p.lde); }
  }
  bool vec = n % 8 == 0 && aligned(p.x, c.size) && aligned(w2) && aligned(p.h, c.size);
  if (c.mode != kPre) {
    vec = vec && aligned(p.y, c.size) && aligned(p.out, c.size) && aligned(w1) && aligned(p.gcol);
    if (c.gate == kElement) vec = vec && aligned(p.gate, c.gate_f32 ? 4 : c.size);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.type == 0 ? forward<__nv_bfloat16>(c.mode, vec, p, s) : c.type == 1 ? forward<__half>(c.mode, vec, p, s)
                                                                               : forward<float>(c.mode, vec, p, s);
}

// Sums of columns in `work` (null: nobody asks): [part_w2 unless kPost][part_c unless kPre], each [groups][n rounded up to 8], and
// part_s [groups] unless kPre.
static void split_work(void* work, int mode, long long groups, int n, float*& w2, float*& c, float*& s) {
  float* at = static_cast<float*>(work);
  w2 = c = s = nullptr;
  if (!at) return;
  const long long size = groups * ((n + 7) / 8 * 8);
  if (mode != kPost) { w2 = at; at += size; }
  if (mode != kPre) { c = at; s = at + size; }
}

// The rows' part of a backward pass: dz (kPre, kPostPre), dy and the gradient of a gate per row or element.  Everything but z, y
// and a gate per row is contiguous.  dout, dy and dgate may be null.  kept: as bshmem_norm_fwd has it; exponents are read by the whole
// 4-byte word that they are in, so up to three bytes behind the last one have to be there.
int bshmem_norm_bwd(int what, const void* dout, const void* dh, const void* z, long long ldz, const void* y, long long ldy, const void* w1,
                    const void* w2, const void* gate, long long ldg, const void* scale, uint64_t scale_bits, const void* rstd, const void* kept,
                    int norms_kept, void* dz, void* dy, void* dgate, void* work, long long rows, int n, void* stream) {
  const Call c(what);
  if (!c.known() || rows < 1 || n < 1 || n > kMaxColumns || rows > 0x7fffffffLL) return refuse_size();
  int groups = 0, sms = 0;
  if (int rc = groups_of(rows, n, &groups)) return rc;
  if (int rc = sm_count(&sms)) return rc;
  BwdParams p = {};
  p.dout = {const_cast<void*>(dout), n};
  p.dh = {const_cast<void*>(dh), n};
  p.z = {const_cast<void*>(z), ldz};
  p.y = {const_cast<void*>(y), ldy};
  p.dz = {dz, n};
  p.dy = {dy, n};
  p.dgate = {dgate, c.gate == kRow ? 1 : n};
  p.w1 = w1; p.w2 = w2;
  p.gate_kind = c.gate;
  if (c.gate == kColumn) p.gcol = gate;
  else p.gate = {const_cast<void*>(gate), ldg};
  p.gcol_f32 = p.gate_f32 = c.gate_f32;
  p.scale = scale; p.scale_f32 = c.scale_f32; p.scale_value = float_of(scale_bits);
  p.w1_f32 = c.w1_f32; p.w2_f32 = c.w2_f32;
  p.rows = rows; p.n = n;
  const float* r = static_cast<const float*>(rstd);
  p.rstd1 = r;
  p.rstd2 = c.mode == kPostPre ? r + rows : r;
  if (c.kept) {
    p.ldq = (n + 15) / 16 * 16;
    p.lde = (n + 127) / 128;
    p.q1 = static_cast<const uint8_t*>(kept);
    p.e1 = p.q1 + norms_kept * rows * p.ldq;
    p.q2 = p.q1 + (c.mode == kPostPre ? rows * p.ldq : 0);
    p.e2 = p.e1 + (c.mode == kPostPre ? rows * p.lde : 0);
  }
  split_work(work, c.mode, groups, n, p.part_w2, p.part_c, p.part_s);
  bool vec = n % 8 == 0;
  if (c.mode != kPost) vec = vec && aligned(p.dh, c.size) && aligned(p.dz, c.size) && aligned(w2) && (c.kept || aligned(p.z, c.size));
  if (c.mode != kPre) {
    vec = vec && aligned(p.dout, c.size) && aligned(p.dy, c.size) && aligned(w1) && aligned(p.gcol) && (c.kept || aligned(p.y, c.size));
    if (c.gate == kElement) vec = vec && aligned(p.gate, c.gate_f32 ? 4 : c.size) && aligned(p.dgate, c.gate_f32 ? 4 : c.size);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Shape shape = backward_shape(rows, n, vec, sms, [&](int chunks) { return backward_words(c.size, c.mode, c.kept, c.gate, c.gate_f32, chunks); },
                                     [&](int chunks) { return backward_held(c.mode, chunks); }, backward_raw(p, c.size));
  return c.type == 0 ? backward<__nv_bfloat16>(c.mode, c.kept, shape, p, s)
         : c.type == 1 ? backward<__half>(c.mode, c.kept, shape, p, s) : backward<float>(c.mode, c.kept, shape, p, s);
}

// The gradients that are sums over rows, of what bshmem_norm_bwd left in `work`; each may be null.
int bshmem_norm_bwd_finish(int what, const void* work, const void* w1, const void* gate, const void* scale, uint64_t scale_bits, void* dw1,
                           void* dw2, void* dgate, void* dscale, long long rows, int n, void* stream) {
  const Call c(what);
  if (!c.known() || rows < 1 || n < 1 || n > kMaxColumns || rows > 0x7fffffffLL) return refuse_size();
  int groups = 0;
  if (int rc = groups_of(rows, n, &groups)) return rc;
  FinishParams f = {};
  float *pw, *pc, *ps;
  split_work(const_cast<void*>(work), c.mode, groups, n, pw, pc, ps);
  f.part_w2 = dw2 ? pw : nullptr;
  f.part_c = dw1 || dgate ? pc : nullptr;
  f.part_s = ps;
  f.w1 = w1;
  f.gcol = c.gate == kColumn ? gate : nullptr;
  f.scale = scale; f.scale_f32 = c.scale_f32; f.scale_value = float_of(scale_bits);
  f.dw1 = dw1; f.dw2 = dw2; f.dgcol = dgate; f.dscale = ps ? dscale : nullptr;
  f.groups = groups; f.n = n;
  f.w1_f32 = c.w1_f32; f.w2_f32 = c.w2_f32; f.gcol_f32 = c.gate_f32;
  const dim3 grid((unsigned)((n + kFinishCols - 1) / kFinishCols)), block(kFinishCols, kFinishLanes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.type == 0 ? launch(norm_bwd_finish_kernel<__nv_bfloat16>, grid, block, 0, f, s)
         : c.type == 1 ? launch(norm_bwd_finish_kernel<__half>, grid, block, 0, f, s) : launch(norm_bwd_finish_kernel<float>, grid, block, 0, f, s);
}

}  // extern "C"
