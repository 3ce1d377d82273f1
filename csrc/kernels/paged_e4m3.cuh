// What the kernels of the e4m3 cache share: code conversions, exponents, rows of packed sequences.
#pragma once
#include <cuda_fp16.h>

#include "paged_e4m3.h"
#include "rb_common.cuh"

namespace rb {

constexpr int kE4LeastExp = -100, kE4MostExp = 119;

// 2^e for e in [-126, 127]
__device__ __forceinline__ float e4_two(int e) { return __int_as_float((e + 127) << 23); }

// The least exponent under which a magnitude (finite, not negative) is at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int e4_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = static_cast<int>(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kE4LeastExp), kE4MostExp);
}
__device__ __forceinline__ float e4_finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;                     // neither infinities nor NaN decide a page's exponent
}

// two numbers to two codes (the first in the low byte): nearest, ties to even, beyond 448 the largest code, NaN stays NaN
__device__ __forceinline__ uint32_t e4_pack2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// two codes to two halves: exact
__device__ __forceinline__ uint32_t e4_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}
// four codes to two pairs of halves
__device__ __forceinline__ void e4_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float2 e4_float2(uint32_t codes) {
  const uint32_t h = e4_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Four codes under an exponent that is larger by `up` (>= 1).  The product is exact in f16 wherever its nearest code is not zero (that
// takes 2^-10 or more, an f16 is exact to 2^-24), and from 19 on every code becomes zero.
__device__ __forceinline__ uint32_t e4_lower4(uint32_t codes, int up) {
  const __half2 f = __half2half2(__float2half(e4_two(-min(up, 24))));
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = e4_half2(codes >> (16 * i));
    const __half2 p = __hmul2(*reinterpret_cast<const __half2*>(&h), f);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&p)));
    out |= static_cast<uint32_t>(r) << (16 * i);
  }
  return out;
}

// The sequence that row r of rows packed one sequence behind the other belongs to: the last b with starts[b] <= r (sequences without rows are
// passed over), found by a whole warp by counting: loads that do not wait for one another.
__device__ __forceinline__ int e4_sequence_of(const int* __restrict__ starts, int batch, int r) {
  int upto = 0;
  for (int i = 1 + (threadIdx.x & 31); i < batch; i += 32) upto += starts[i] <= r ? 1 : 0;
  return __reduce_add_sync(0xffffffffu, upto);
}

// Page `i` of sequence b, -1 where the table has none or names one that is not there.
__device__ __forceinline__ int e4_page(const int* __restrict__ tables, int max_blocks, long long num_blocks, int b, int i) {
  if (i < 0 || i >= max_blocks) return -1;
  const int p = tables[static_cast<long long>(b) * max_blocks + i];
  return p < 0 || p >= num_blocks ? -1 : p;
}

// Eight numbers of a row.  `largest` takes the larger magnitudes of eight into `acc` as their bits, two 16-bit ones beside each other; `one` makes one number's
// bits of that, `value` the number; from kNotFinite on they are an infinity's or a NaN's.
template <typename T>
struct E4Row;
__device__ __forceinline__ void e4_largest16(const uint4& u, uint32_t& acc) {
  acc = __vmaxu2(__vmaxu2(acc, u.x & 0x7fff7fffu), u.y & 0x7fff7fffu);
  acc = __vmaxu2(__vmaxu2(acc, u.z & 0x7fff7fffu), u.w & 0x7fff7fffu);
}
template <>
struct E4Row<__nv_bfloat16> {
  static constexpr uint32_t kNotFinite = 0x7f80u;
  static __device__ __forceinline__ void largest(const uint4 (&raw)[1], uint32_t& acc) { e4_largest16(raw[0], acc); }
  static __device__ __forceinline__ uint32_t one(uint32_t acc) { return max(acc & 0xffffu, acc >> 16); }
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u[1] = {*reinterpret_cast<const uint4*>(p)};
    of(u, x);
  }
  static __device__ __forceinline__ void of(const uint4 (&raw)[1], float (&x)[8]) {
    const uint4 u = raw[0];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct E4Row<__half> {
  static constexpr uint32_t kNotFinite = 0x7c00u;
  static __device__ __forceinline__ void largest(const uint4 (&raw)[1], uint32_t& acc) { e4_largest16(raw[0], acc); }
  static __device__ __forceinline__ uint32_t one(uint32_t acc) { return max(acc & 0xffffu, acc >> 16); }
  static __device__ __forceinline__ float value(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
  static __device__ __forceinline__ void load(const __half* p, float (&x)[8]) {
    const uint4 u[1] = {*reinterpret_cast<const uint4*>(p)};
    of(u, x);
  }
  static __device__ __forceinline__ void of(const uint4 (&raw)[1], float (&x)[8]) {
    const uint4 u = raw[0];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__half* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct E4Row<float> {
  static constexpr uint32_t kNotFinite = 0x7f800000u;
  static __device__ __forceinline__ void largest(const uint4 (&raw)[2], uint32_t& acc) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      acc = max(acc, max(max(raw[i].x & 0x7fffffffu, raw[i].y & 0x7fffffffu), max(raw[i].z & 0x7fffffffu, raw[i].w & 0x7fffffffu)));
  }
  static __device__ __forceinline__ uint32_t one(uint32_t acc) { return acc; }
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits); }
  static __device__ __forceinline__ void load(const float* p, float (&x)[8]) {
    const uint4 u[2] = {reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]};
    of(u, x);
  }
  static __device__ __forceinline__ void of(const uint4 (&raw)[2], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[4 * i] = __uint_as_float(raw[i].x);
      x[4 * i + 1] = __uint_as_float(raw[i].y);
      x[4 * i + 2] = __uint_as_float(raw[i].z);
      x[4 * i + 3] = __uint_as_float(raw[i].w);
    }
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
};

}  // namespace rb

namespace rbhost {
// 0 where the pages are as paged_e4m3.h says
inline int e4_check(const RbPagesE4m3& p) {
  if (!p.k || !p.v || !p.k_exp || !p.v_exp || p.num_blocks <= 0 || p.num_blocks > 0x7fffffffll || p.block_size <= 0 || (p.block_size & 15) ||
      p.block_size > 1 << 20 || p.kv_heads <= 0 ||
      (p.head_dim != 64 && p.head_dim != 128))
    return -1;
  if ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) return -2;
  return 0;
}
}  // namespace rbhost
