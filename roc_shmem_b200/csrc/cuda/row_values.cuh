// row_values.cuh — eight neighbouring values of a row: loads, stores and conversion of bf16, fp16 and fp32, the 8-bit form in
// which activations are kept between the forward and the backward pass, and sums over the threads of a row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstring>

namespace bshmem {
namespace rows {

// ---- conversion ---------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// ---- two fp32 values at a time -------------------------------------------------------------------
// One instruction for two: these kernels issue more than they wait for.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Eight neighbouring values, as pairs.
struct Vals {
  float2 p[4];
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = both(v);
  }
};

// Eight values as they lie in memory: one 16-byte word of a 2-byte type, two of fp32.
template <typename T> struct alignas(16) Raw8 {
  static constexpr int kWords = sizeof(T) / 2;
  T v[8];
  __device__ __forceinline__ void set(int i, uint4 w) { memcpy(reinterpret_cast<char*>(v) + 16 * i, &w, 16); }
  __device__ __forceinline__ uint4 get(int i) const {
    uint4 w;
    memcpy(&w, reinterpret_cast<const char*>(v) + 16 * i, 16);
    return w;
  }
};

template <typename T> __device__ __forceinline__ Vals unpack(const Raw8<T>& r) {
  Vals v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.p[i] = make_float2(to_float<T>(r.v[2 * i]), to_float<T>(r.v[2 * i + 1]));
  return v;
}
template <> __device__ __forceinline__ Vals unpack(const Raw8<__nv_bfloat16>& r) {      // a bf16 is the high half of its fp32
  Vals v;
  const uint4 w = r.get(0);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v.p[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  return v;
}
template <> __device__ __forceinline__ Vals unpack(const Raw8<__half>& r) {
  Vals v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.p[i] = __half22float2(__halves2half2(r.v[2 * i], r.v[2 * i + 1]));
  return v;
}
template <typename T> __device__ __forceinline__ Raw8<T> pack(const Vals& v) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) { r.v[2 * i] = from_float<T>(v.p[i].x); r.v[2 * i + 1] = from_float<T>(v.p[i].y); }
  return r;
}
template <> __device__ __forceinline__ Raw8<__nv_bfloat16> pack(const Vals& v) {
  Raw8<__nv_bfloat16> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 t = __float22bfloat162_rn(v.p[i]);
    r.v[2 * i] = t.x; r.v[2 * i + 1] = t.y;
  }
  return r;
}
template <> __device__ __forceinline__ Raw8<__half> pack(const Vals& v) {
  Raw8<__half> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 t = __float22half2_rn(v.p[i]);
    r.v[2 * i] = __low2half(t); r.v[2 * i + 1] = __high2half(t);
  }
  return r;
}

// How eight values lie in a row.  kVector: columns col .. col + 7, the row is 16-byte aligned and the row's length n % 8 == 0.  kSingle:
// the same columns, one by one.  kStrided: one by one too, but for a warp on 256 neighbouring columns the lanes' j-th values are
// neighbours (lane, lane + 32, ...), so that each access of the warp is whole sectors.
enum Access : int { kSingle = 0, kVector = 1, kStrided = 2 };
template <int kAccess> __device__ __forceinline__ int column_of(int col, int j) {
  return kAccess == kStrided ? (col & ~255) + (col >> 3 & 31) + 32 * j : col + j;
}
// Columns from n on are zeros.  Plain loads: a kernel that starts while the one before still writes its operands may not say that they are read
// only, or the compiler could move a load in front of the wait for that kernel.
template <int kAccess, typename T> __device__ __forceinline__ Raw8<T> load8(const T* row, int col, int n) {
  Raw8<T> r;
  if constexpr (kAccess == kVector) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords; ++i) r.set(i, col < n ? reinterpret_cast<const uint4*>(row + col)[i] : make_uint4(0, 0, 0, 0));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = column_of<kAccess>(col, j) < n ? row[column_of<kAccess>(col, j)] : from_float<T>(0.f);
  }
  return r;
}
template <int kAccess, typename T> __device__ __forceinline__ void store8(T* row, int col, int n, const Raw8<T>& r) {
  if constexpr (kAccess == kVector) {
    if (col < n) {
#pragma unroll
      for (int i = 0; i < Raw8<T>::kWords; ++i) reinterpret_cast<uint4*>(row + col)[i] = r.get(i);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (column_of<kAccess>(col, j) < n) row[column_of<kAccess>(col, j)] = r.v[j];
  }
}

// A vector over the columns (a weight, a gate per channel) in the rows' own type T or in fp32; ones where there is none.
template <int kAccess, typename T> __device__ __forceinline__ Vals vector8(const void* vec, bool f32, int col, int n) {
  Vals v;
  if (!vec) v.fill(1.f);
  else if (f32) v = unpack(load8<kAccess>(static_cast<const float*>(vec), col, n));
  else v = unpack(load8<kAccess>(static_cast<const T*>(vec), col, n));
  return v;
}

// ---- activations in 8 bits -------------------------------------------------------------------------
// e4m3 times one power of two for each row and 128 columns, the smallest that holds the block's largest finite value (448 is
// e4m3's largest): a power of two loses nothing, neither here nor on the way back, and it is one byte (exponent + 127).
// Infinities come back as NaN; e4m3 has none.
__device__ __forceinline__ float block_scale_bits(uint32_t e) { return __uint_as_float(e << 23); }
// The largest exponent byte of a type's blocks.  Only there could a value round up to a power of two that the type does not have
// (2^128, 2^16 for fp16): such values stay at 240 steps instead of 256.
template <typename T> constexpr uint32_t kTopExponent = 247;
template <> constexpr uint32_t kTopExponent<__half> = 135;

// The eight bytes of a lane's values; kAny: some may be no numbers, or so large that they could round up (see kTopExponent).
template <typename T, bool kAny> __device__ __forceinline__ uint2 bytes8(const Vals& v, uint32_t e) {
  const float2 down = both(block_scale_bits(254u - e));
  const float most = e == kTopExponent<T> ? 240.f : 448.f;
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint16_t two[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 given = v.p[2 * h + i];
      float2 f = mul2(given, down);                   // subnormal numbers count: no .ftz
      if constexpr (kAny) f = make_float2(fminf(fmaxf(f.x, -most), most), fminf(fmaxf(f.y, -most), most));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two[i]) : "f"(f.y), "f"(f.x));
      if constexpr (kAny) {                           // the limits made a number of what is none
        if ((__float_as_uint(given.x) & 0x7fffffffu) >= 0x7f800000u) two[i] |= 0x7f;
        if ((__float_as_uint(given.y) & 0x7fffffffu) >= 0x7f800000u) two[i] |= 0x7f00;
      }
    }
    out[h] = two[0] | (uint32_t)two[1] << 16;
  }
  return make_uint2(out[0], out[1]);
}
// largest = m * 2^(E - 127), m in [1, 2), and 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t exponent_byte(uint32_t largest) {
  return (uint32_t)max((int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u), 1);
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t a = __float_as_uint(v) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
// All 32 lanes take part; 16 / kEach neighbours hold a block, kEach eights of it each.  The bytes of this lane's values, which are of type T, and
// the block's exponent byte.
template <typename T, int kEach> __device__ __forceinline__ void encode(const Vals (&v)[kEach], uint2 (&q)[kEach], uint32_t& e) {
  float top = 0.f;
  float2 odd = both(0.f);                             // NaN if one of the values is no number, or infinite
#pragma unroll
  for (int k = 0; k < kEach; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top = fmaxf(top, fmaxf(fabsf(v[k].p[i].x), fabsf(v[k].p[i].y)));
      odd = fma2(v[k].p[i], both(0.f), odd);
    }
  uint32_t bits = __float_as_uint(top);
  // rare, and then for the whole warp: the largest of the finite values, and the careful conversion
  const bool any = __any_sync(0xffffffffu, odd.x + odd.y != 0.f || bits >= (kTopExponent<T> + 7u) << 23);
  if (any) {
    bits = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) bits = max(bits, max(finite_bits(v[k].p[i].x), finite_bits(v[k].p[i].y)));
  }
#pragma unroll
  for (int o = 8 / kEach; o; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  e = exponent_byte(bits);
#pragma unroll
  for (int k = 0; k < kEach; ++k) q[k] = any ? bytes8<T, true>(v[k], e) : bytes8<T, false>(v[k], e);
}
template <typename T> __device__ __forceinline__ uint2 encode8(const Vals& v, uint32_t& e) {
  uint2 q[1];
  encode<T, 1>({v}, q, e);
  return q[0];
}
__device__ __forceinline__ Vals decode8(uint2 q, uint32_t e) {
  Vals v;
  const float up = block_scale_bits(e);
  const uint32_t w[2] = {q.x, q.y};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t two;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((uint16_t)(w[h] >> (16 * i))));
      __half2 pair;
      memcpy(&pair, &two, 4);
      const float2 f = __half22float2(pair);
      v.p[2 * h + i] = mul2(f, both(up));             // subnormal numbers count: no .ftz
    }
  return v;
}

// Columns of a row of bytes: those behind the n that have values are zeros.
__device__ __forceinline__ int byte_columns(int n) { return (n + 15) & ~15; }
// A lane's eight values into a row of bytes and exponents, and back.  kStrided: the warp's 256 columns are two blocks, of the lanes'
// first four and last four values.
template <int kAccess, typename T> __device__ __forceinline__ void keep8(uint8_t* q, uint8_t* e, int col, int n, const Vals& v) {
  if constexpr (kAccess == kVector) {
    uint32_t x;
    const uint2 b = encode8<T>(v, x);
    if (col < byte_columns(n)) *reinterpret_cast<uint2*>(q + col) = b;
    if (col < n && col % 128 == 0) e[col / 128] = (uint8_t)x;
  } else {
    uint32_t x[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i / 2] = max(x[i / 2], max(finite_bits(v.p[i].x), finite_bits(v.p[i].y)));
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      x[0] = max(x[0], __shfl_xor_sync(0xffffffffu, x[0], o));
      x[1] = max(x[1], __shfl_xor_sync(0xffffffffu, x[1], o));
    }
    const uint32_t e0 = exponent_byte(x[0]), e1 = exponent_byte(x[1]), low = bytes8<T, true>(v, e0).x, high = bytes8<T, true>(v, e1).y;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (column_of<kAccess>(col, j) < byte_columns(n)) q[column_of<kAccess>(col, j)] = (uint8_t)((j < 4 ? low : high) >> (8 * (j & 3)));
    if (col % 256 == 0) {
      if (col < n) e[col / 128] = (uint8_t)e0;
      if (col + 128 < n) e[col / 128 + 1] = (uint8_t)e1;
    }
  }
}
template <int kAccess> __device__ __forceinline__ Vals kept8(const uint8_t* q, const uint8_t* e, int col, int n) {
  if constexpr (kAccess == kVector) {
    uint2 b = make_uint2(0, 0);
    uint32_t x = 1;
    if (col < n) {
      b = *reinterpret_cast<const uint2*>(q + col);
      x = e[col / 128];
    }
    return decode8(b, x);
  } else {
    const int block = (col & ~255) / 128;
    const uint32_t e0 = col - (col & 255) < n ? e[block] : 1, e1 = col - (col & 255) + 128 < n ? e[block + 1] : 1;
    uint2 b = make_uint2(0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = column_of<kAccess>(col, j) < n ? q[column_of<kAccess>(col, j)] : 0;
      if (j < 4) b.x |= x << (8 * j);
      else b.y |= x << (8 * (j - 4));
    }
    const Vals low = decode8(b, e0), high = decode8(b, e1);
    Vals v;
    v.p[0] = low.p[0]; v.p[1] = low.p[1]; v.p[2] = high.p[2]; v.p[3] = high.p[3];
    return v;
  }
}

// ---- sums over a row -----------------------------------------------------------------------------------
// blockDim.x threads (whole warps) work on one row, blockDim.y rows on a block.  One barrier per sum: the words of two
// sums in a row differ, so a warp that is ahead writes where nobody reads any more.
constexpr int kMaxWarps = 32;
struct RowSum {
  float* words;                                       // [2][kMaxWarps], shared
  int turn = 0;
  __device__ __forceinline__ explicit RowSum(float* w) : words(w) {}
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1) return v;
    float* mine = words + turn * kMaxWarps + threadIdx.y * warps;
    turn ^= 1;
    if (lane == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? mine[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
};

}  // namespace rows
}  // namespace bshmem
