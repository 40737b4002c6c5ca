// Conversions between values and the 8-bit codes of the KV cache.
//
// A code c of a block whose scale byte is u stands for c * 2^(u - 127) (E8M0
// scales).  u is the smallest byte >= 1 with amax <= qmax * 2^(u - 127); 255
// marks an int8 block that was given a non-finite value and reads as NaN.  The
// scales are powers of two so that a block whose scale grows while tokens are
// appended keeps its e4m3 codes exactly (only codes that leave the normal range
// round again), and so that applying one is an exponent shift.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "dta_cache.h"

namespace dta {

// 2^(u - 127) for a scale byte; u = 0 (a block nothing was written to) is 2^-127.
__device__ __forceinline__ float cache_scale(int u) {
  return u == 0 ? __uint_as_float(0x00400000u) : u == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)u << 23);
}
// 2^(127 - u), the factor that a written value is multiplied by (1 <= u <= 253).
__device__ __forceinline__ float cache_inv_scale(int u) { return __uint_as_float((uint32_t)(254 - u) << 23); }

// Scale byte that a block with this largest finite magnitude needs.  With
// amax = m * 2^E, 1 <= m < 2, and qmax = Q * 2^K: u - 127 = E - K, or one more
// when m > Q.  Subnormal amax fall below the least scale (u = 1) by themselves.
template <int FMT>
__device__ __forceinline__ int cache_need(float amax) {
  constexpr uint32_t kMant = FMT == CACHE_E4M3 ? 0x600000u : 0x7e0000u;  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr int kExp = FMT == CACHE_E4M3 ? 8 : 6;
  const uint32_t bits = __float_as_uint(amax);
  const int u = (int)(bits >> 23) - kExp + ((bits & 0x7fffffu) > kMant ? 1 : 0);
  return max(u, 1);
}

// a * b elementwise (one instruction for two products).
__device__ __forceinline__ float2 mul2(float2 a, float b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b));
  return r;
}

// Four finite values times a power of two -> four codes (value 0 in the low byte),
// ties to even; the products lie within the format.
template <int FMT>
__device__ __forceinline__ uint32_t cache_pack4(float2 a, float2 b, float inv) {
  if constexpr (FMT == CACHE_E4M3) {
    a = mul2(a, inv);
    b = mul2(b, inv);
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  } else {
    // x * inv is exact, so x * inv + 1.5 * 2^23 rounds it once, to an integer in the low bits
    const float magic = 12582912.f;
    const uint32_t x = __float_as_uint(fmaf(a.x, inv, magic)), y = __float_as_uint(fmaf(a.y, inv, magic));
    const uint32_t z = __float_as_uint(fmaf(b.x, inv, magic)), w = __float_as_uint(fmaf(b.y, inv, magic));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  }
}

// Two codes in the low (HI = 0) or high half of `w` -> two fp16 values (exact).
template <int FMT, int HI>
__device__ __forceinline__ uint32_t cache_half2(uint32_t w) {
  uint32_t r;
  if constexpr (FMT == CACHE_E4M3) {
    const uint16_t h = (uint16_t)(HI ? w >> 16 : w & 0xffffu);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  } else {
    // w holds code + 128 per byte: the byte under 0x64 is fp16 1024 + 128 + code
    const uint32_t x = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  }
  return r;
}
// What cache_half2 expects: e4m3 codes as they are, int8 codes with 128 added.
template <int FMT>
__device__ __forceinline__ uint32_t cache_bias(uint32_t w) {
  return FMT == CACHE_INT8 ? w ^ 0x80808080u : w;
}

// Four codes -> four fp32 values (unscaled).
template <int FMT>
__device__ __forceinline__ void cache_unpack4(uint32_t w, float (&f)[4]) {
  const uint32_t b = cache_bias<FMT>(w);
  const uint32_t lo = cache_half2<FMT, 0>(b), hi = cache_half2<FMT, 1>(b);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}

}  // namespace dta
