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
  return u == 0     ? __uint_as_float(0x00400000u)
         : u == 255 ? __uint_as_float(0x7fc00000u)
                    : __uint_as_float((uint32_t)u << 23);
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

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// Two values -> two e4m3 codes, ties to even.
__device__ __forceinline__ uint32_t e4m3_pack2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// Four finite values times a power of two -> four codes (value 0 in the low byte),
// ties to even; the products lie within the format.
template <int FMT>
__device__ __forceinline__ uint32_t cache_pack4(float2 a, float2 b, float inv) {
  if constexpr (FMT == CACHE_E4M3) {
    a = mul2(a, make_float2(inv, inv));
    b = mul2(b, make_float2(inv, inv));
    return e4m3_pack2(a.x, a.y) | (e4m3_pack2(b.x, b.y) << 16);
  } else {
    // x * inv is exact, so x * inv + 1.5 * 2^23 rounds it once, to an integer in the low bits
    const float magic = 12582912.f;
    const uint32_t x = __float_as_uint(fmaf(a.x, inv, magic)), y = __float_as_uint(fmaf(a.y, inv, magic));
    const uint32_t z = __float_as_uint(fmaf(b.x, inv, magic)), w = __float_as_uint(fmaf(b.y, inv, magic));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  }
}

__device__ __forceinline__ uint32_t e4m3_half2(uint16_t h) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  return r;
}
// int8 codes in bytes 0 and 2 -> two fp16: the byte code + 128 under 0x64 is 1024 + 128 + code.
__device__ __forceinline__ uint32_t int8_half2(uint32_t w) {
  uint32_t r = (w & 0x00ff00ffu) ^ 0x64806480u;
  asm("sub.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));
  return r;
}
// Four codes of each of two rows -> four fp16 pairs (row a's code i, row b's code i), exact.
template <int FMT>
__device__ __forceinline__ void cache_zip(uint32_t a, uint32_t b, uint32_t (&o)[4]) {
  if constexpr (FMT == CACHE_E4M3) {
    const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
    o[0] = e4m3_half2((uint16_t)(x & 0xffffu));
    o[1] = e4m3_half2((uint16_t)(x >> 16));
    o[2] = e4m3_half2((uint16_t)(y & 0xffffu));
    o[3] = e4m3_half2((uint16_t)(y >> 16));
  } else {
    const uint32_t x = __byte_perm(a, b, 0x5410), y = __byte_perm(a, b, 0x7632);
    o[0] = int8_half2(x);
    o[1] = int8_half2(x >> 8);
    o[2] = int8_half2(y);
    o[3] = int8_half2(y >> 8);
  }
}

// Four codes -> four fp32 values (unscaled).
template <int FMT>
__device__ __forceinline__ void cache_unpack4(uint32_t w, float (&f)[4]) {
  if constexpr (FMT == CACHE_E4M3) {
    const uint32_t lo = e4m3_half2((uint16_t)(w & 0xffffu)), hi = e4m3_half2((uint16_t)(w >> 16));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
  } else {
    // code + 128 in the low byte under 2^23: an fp32 integer
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)) - (8388608.f + 128.f);
  }
}

}  // namespace dta
