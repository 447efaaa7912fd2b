// gemm_w4.cu — linear layers with weights of 4 bits: entry points, the quantiser, and the weights in bf16 for products with many
// tokens.  q: [N, K/2] bytes, the low half of a byte is the column of even number; s, z: [N, K/group].  The products with few
// tokens are in w4_stream.cuh.
#include <atomic>

#include "w4_stream.cuh"

using namespace bshmem;

namespace {

// w in bf16, for products with many tokens on the bf16 kernels: each weight is rounded once (2^-8 of itself at most), as a layer
// that keeps its weights in bf16 has them.  A thread has four words of eight columns, a block's width apart.
struct WidenParams {
  const uint32_t* q;
  const __nv_bfloat16* s;
  const uint8_t* z;
  __nv_bfloat16* w;
  long long words;                                    // N * K / 8
  int per_group;                                      // words of a group; K is whole groups, so rows need no looking at
};
constexpr int kWidenWords = 4;
__global__ void __launch_bounds__(256) w4_widen_kernel(const WidenParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long first = (long long)blockIdx.x * (256 * kWidenWords) + threadIdx.x;
  uint32_t w[kWidenWords], z[kWidenWords];
  __nv_bfloat16 s[kWidenWords];
#pragma unroll
  for (int j = 0; j < kWidenWords; ++j) {
    const long long i = min(first + j * 256, p.words - 1), g = i / p.per_group;
    w[j] = p.q[i];
    s[j] = p.s[g];
    z[j] = p.z ? p.z[g] : 8;
  }
#pragma unroll
  for (int j = 0; j < kWidenWords; ++j) {
    uint32_t o[4];                                    // (0, 4) (1, 5) (2, 6) (3, 7)
    w4::widen(w[j], w4::as_pair(0x43004300u | z[j] | z[j] << 16), o);
    // a product of bf16 values rounded once is the weight rounded once: q - z is exact
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = w4::as_word(__hmul2(w4::as_pair(o[k]), __bfloat162bfloat162(s[j])));
    if (first + j * 256 < p.words)
      ptx::st_v4(p.w + (first + j * 256) * 8, make_uint4(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410),
                                                         __byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632)));
  }
}

// bf16 weights to 4 bits; a warp has a group.  Without zero points the scale is (largest magnitude) / 7, with them
// (largest - smallest) / 15 of a range that has zero in it, rounded to bf16; q is the nearest of what that can say.  A group with an
// infinity or a NaN has no scale: it gets NaN, and so all of its weights are.
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
  bool odd = false;                                   // the minimum and the maximum pass over a NaN
  for (int k = lane; k < p.group; k += 32) {
    const float v = __bfloat162float(w[k]);
    odd |= (__float_as_uint(v) & 0x7fffffffu) >= 0x7f800000u;
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
  odd = __any_sync(0xffffffffu, odd);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // a range that fp32 does not hold is fifteen parts all the same
  const float range = hi - lo, part = range <= 3.4028234e38f ? __fdiv_rn(range, 15.f) : __fdiv_rn(hi, 15.f) + __fdiv_rn(-lo, 15.f);
  const __nv_bfloat16 sb = odd ? __ushort_as_bfloat16(0x7fff) : __float2bfloat16_rn(p.z ? part : __fdiv_rn(fmaxf(hi, -lo), 7.f));
  const float s = odd ? 0.f : __bfloat162float(sb);
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

template <typename K, typename P>
int launch(K* kernel, dim3 grid, int threads, int cluster, int shared, const P& p, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
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

// How many clusters of `size` blocks the device holds at once, one block per SM (clusters do not span GPCs).
int resident(void (*kernel)(w4::Params), int dev, int size, int threads, int sms) {
  static std::atomic<int> cache[64][9];               // racing threads write the same number; every form takes a whole SM
  std::atomic<int>& slot = cache[dev][size];
  int n = slot.load(std::memory_order_relaxed);
  if (n) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(size * sms));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = w4::SMEM_BYTES;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = sms / size; }
  slot.store(n, std::memory_order_relaxed);
  return n;
}

template <int kNt, int kSubs> int stream_product(w4::Params& p, int sms, void* stream) {
  int dev = 0;
  BSHMEM_CUDA_TRY(cudaGetDevice(&dev));
  static std::atomic<bool> prepared[64];
  if (!prepared[dev].load(std::memory_order_relaxed)) {
    BSHMEM_CUDA_TRY(cudaFuncSetAttribute(w4::w4_stream_kernel<kNt, kSubs>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)w4::SMEM_BYTES));
    prepared[dev].store(true, std::memory_order_relaxed);
  }
  int rc = host::make_tmap_2d(&p.map_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.x, p.T, p.K, p.ldx, kNt, 64);
  if (rc) return rc;
  // Split the columns so that the longest block is shortest, in stages; adding the parts up costs about two.
  const int kb = (p.K + 2 * w4::BK - 1) / (2 * w4::BK), chunks = (p.T + kNt - 1) / kNt;
  const long long tiles = (long long)((p.N + w4::ROWS - 1) / w4::ROWS) * chunks;
  long long best = 0;
  for (int s = 1; s <= 8; ++s) {
    const long long at_once = resident(w4::w4_stream_kernel<kNt, kSubs>, dev, s, w4::threads(kNt, kSubs), sms);
    const long long cost = (tiles + at_once - 1) / at_once * ((kb + s - 1) / s) + (s > 1 ? 2 : 0);
    if (s == 1 || cost < best) { best = cost; p.split = s; }
  }
  return launch(w4::w4_stream_kernel<kNt, kSubs>, dim3((unsigned)((p.N + w4::ROWS - 1) / w4::ROWS * p.split), (unsigned)chunks), w4::threads(kNt, kSubs), p.split,
                w4::SMEM_BYTES, p, stream);
}
template <int kNt> int stream_groups(w4::Params& p, int sms, void* stream) {
  // four groups of 64 tokens, twice, would be more than tensor memory has
  if (p.group == 32) return stream_product<kNt == 64 ? 32 : kNt, 4>(p, sms, stream);
  return p.group == 64 ? stream_product<kNt, 2>(p, sms, stream) : stream_product<kNt, 1>(p, sms, stream);
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
                  void* stream, int timeout_ms) {
  if (!shape_ok(N, K, group)) return 1;
  if (ldx % 8 || !aligned(x) || !aligned(q) || T > 65535 * 16) { host::last_error() = "w4: needs 16-byte aligned x and q, row pitch % 8 == 0"; return 1; }
  if (T <= 0) return 0;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  w4::Params p;
  p.x = x; p.ldx = ldx;
  p.s = static_cast<const __nv_bfloat16*>(s);
  p.z = static_cast<const uint8_t*>(z);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = N;
  p.T = T; p.N = N; p.K = K; p.group = group;
  p.timeout_ns = (unsigned long long)(timeout_ms > 0 ? timeout_ms : 2000) * 1000000ull;
  if (int rc = host::make_tmap_2d(&p.map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, N, K / 2, K / 2, w4::ROWS, w4::BK)) return rc;
  return T <= 16 ? stream_groups<16>(p, sms, stream) : T <= 32 ? stream_groups<32>(p, sms, stream) : stream_groups<64>(p, sms, stream);
}

// 0 if no in-kernel bounded wait ran out on the current device since the last clear, else the site code; synchronises.
int bshmem_w4_error_site(int clear) {
  int site = -1, zero = 0;
  if (cudaMemcpyFromSymbol(&site, w4::error_word, sizeof(int)) != cudaSuccess) return -1;
  if (clear && site && cudaMemcpyToSymbol(w4::error_word, &zero, sizeof(int)) != cudaSuccess) return -1;
  return site;
}

// w [N, K] bf16 contiguous and 16-byte aligned.
int bshmem_w4_widen(const void* q, const void* s, const void* z, void* w, int N, int K, int group, void* stream) {
  if (!shape_ok(N, K, group)) return 1;
  if (!aligned(q) || !aligned(w)) { host::last_error() = "w4: needs 16-byte aligned q and w"; return 1; }
  const WidenParams p = {static_cast<const uint32_t*>(q), static_cast<const __nv_bfloat16*>(s), static_cast<const uint8_t*>(z),
                         static_cast<__nv_bfloat16*>(w), (long long)N * (K / 8), group / 8};
  const long long blocks = (p.words + 256 * kWidenWords - 1) / (256 * kWidenWords);
  if (blocks > 0x7fffffffLL) { host::last_error() = "w4: matrix too large"; return 1; }
  return launch(w4_widen_kernel, dim3((unsigned)blocks), 256, 1, 0, p, stream);
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
