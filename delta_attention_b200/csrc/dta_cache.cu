// Writing an 8-bit KV cache and reading it back (sm_100a).
//
// Write: CTA = one scale block of one head of K or V.  It loads the block's new
// rows once into registers, reduces their largest finite magnitude, and stores
// the codes; a block that already holds earlier tokens keeps the larger of its
// own and the new scale, and where that raises the scale the CTA rounds the
// earlier codes to it.  Every scale block belongs to one CTA, so nothing is
// shared between CTAs.  Read: codes times their block's scale, rounded once.
// Both are streams: their bound is the memory traffic.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "dta_cache.h"
#include "dta_cache_codes.cuh"
#include "dta_ptx.cuh"

namespace dta {

// Largest of the unsigned 16-bit halves.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight consecutive elements of a source row.  Magnitudes compare as the integers
// that their bits are (infinities and NaN above all finite values): `top` folds the
// row's bits into a running maximum, `bits` turns that into the bits of an fp32.
template <int SRC>
struct Row8;
template <>
struct Row8<CACHE_BF16> {
  uint4 r;
  __device__ __forceinline__ void load(const void* base, long long off) {
    r = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + off);
  }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = max_u16x2(max_u16x2(m, r.x & 0x7fff7fffu), r.y & 0x7fff7fffu);
    m = max_u16x2(max_u16x2(m, r.z & 0x7fff7fffu), r.w & 0x7fff7fffu);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return max(m & 0xffffu, m >> 16) << 16; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Row8<CACHE_FP16> {
  uint4 r;
  __device__ __forceinline__ void load(const void* base, long long off) {
    r = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + off);
  }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = max_u16x2(max_u16x2(m, r.x & 0x7fff7fffu), r.y & 0x7fff7fffu);
    m = max_u16x2(max_u16x2(m, r.z & 0x7fff7fffu), r.w & 0x7fff7fffu);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
};
template <>
struct Row8<CACHE_FP32> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* base, long long off) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + off);
    a = p[0];
    b = p[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void top(uint32_t& m) const {
    float f[8];
    get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return m; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

// Largest value over the CTA; its words may be reused after the next barrier.
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  __shared__ uint32_t red[16];
  v = __reduce_max_sync(0xffffffffu, v);
  if (blockDim.x == 32) {
    __syncwarp();
    return v;
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v = max(v, red[w]);
  return v;
}

constexpr int WRITE_CHUNKS = 4;  // 8-element chunks per thread: T * d / 32 threads, at most 512

template <int HD, int FMT, int SRC>
__global__ void __launch_bounds__(512) cache_write_kernel(const __grid_constant__ CacheWriteParams p) {
  constexpr int RC = HD / 8;  // chunks per row
  const int b = blockIdx.y / p.Hkv, h = blockIdx.y - b * p.Hkv;
  const int side = blockIdx.z;
  const CacheSide& S = p.side[side];
  // [first, end): the positions that this call writes in sequence b
  const int pos = p.pos_dev ? p.pos_dev[b * p.pos_step] : p.pos;
  const int len = p.lengths ? p.lengths[b * p.len_step] : p.n_new;
  int first = pos, end = pos + min(max(len, 0), p.n_new);
  if (pos < 0 || pos > p.capacity || len < 0 || len > p.n_new || end > p.capacity) {
    // a device position or length outside the cache: nothing of this sequence is written
    if (threadIdx.x == 0 && blockIdx.x == 0 && p.error_word) atomicCAS(p.error_word, 0, (int)KERR_BAD_ROW);
    return;
  }
  const int blk = (first >> p.log_block) + blockIdx.x;
  const int lo = blk << p.log_block;
  if (lo >= end) return;  // (also every block of an empty sequence, whose end is first)
  if (first == end) return;

  const long long src0 = (long long)b * p.src_sb[side] + (long long)h * p.src_sh[side];
  uint8_t* codes = S.codes + (long long)b * S.sb + (long long)h * S.sh;
  uint8_t* scale = S.scale + (long long)b * S.scale_sb + (long long)h * S.scale_sh + blk;
  Row8<SRC> x[WRITE_CHUNKS];
#pragma unroll
  for (int c = 0; c < WRITE_CHUNKS; ++c) {
    const int idx = c * blockDim.x + threadIdx.x;
    const int t = lo + idx / RC;
    if (t >= first && t < end) x[c].load(p.src[side], src0 + (long long)(t - first) * p.src_ss[side] + (idx % RC) * 8);
    else x[c].zero();
  }
  const bool held = lo < first;  // the block holds tokens before this call's first
  const int u_old = held ? *scale : 0;
  uint32_t amax = 0;  // bits of the largest magnitude
#pragma unroll
  for (int c = 0; c < WRITE_CHUNKS; ++c) x[c].top(amax);
  amax = block_max(Row8<SRC>::bits(amax));
  const bool finite = amax < 0x7f800000u;
  if (!finite && FMT == CACHE_E4M3) {  // the scale goes by the finite values
    amax = 0;
#pragma unroll
    for (int c = 0; c < WRITE_CHUNKS; ++c) {
      float f[8];
      x[c].get(f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(f[i]) & 0x7fffffffu;
        if (a < 0x7f800000u) amax = max(amax, a);
      }
    }
    __syncthreads();  // block_max's words are read
    amax = block_max(amax);
  }
  // (block_max's barrier comes after every thread's read of the old scale)
  const int u = max(amax >= 0x7f800000u ? 255 : cache_need<FMT>(__uint_as_float(amax)), u_old);
  if (threadIdx.x == 0) *scale = (uint8_t)u;
  const float inv = u == 255 ? 0.f : cache_inv_scale(u);
#pragma unroll
  for (int c = 0; c < WRITE_CHUNKS; ++c) {
    const int idx = c * blockDim.x + threadIdx.x;
    const int t = lo + idx / RC;
    if (t < first || t >= end) continue;
    float f[8];
    x[c].get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // e4m3 has no infinity: a non-finite value becomes NaN
      if (FMT == CACHE_E4M3 && !finite && (__float_as_uint(f[i]) & 0x7fffffffu) >= 0x7f800000u)
        f[i] = __uint_as_float(0x7fc00000u);
      f[i] *= inv;
    }
    *reinterpret_cast<uint2*>(codes + (long long)t * S.ss + (idx % RC) * 8) =
        make_uint2(cache_pack4<FMT>(f[0], f[1], f[2], f[3]), cache_pack4<FMT>(f[4], f[5], f[6], f[7]));
  }
  if (!held || u == u_old) return;
  // the scale rose: the block's earlier codes are rounded to it
  const float shrink = u - u_old > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (u - u_old)) << 23);
  for (int idx = threadIdx.x; idx < (first - lo) * RC; idx += blockDim.x) {
    uint2* dst = reinterpret_cast<uint2*>(codes + (long long)(lo + idx / RC) * S.ss + (idx % RC) * 8);
    const uint2 w = *dst;
    float f[4], g[4];
    cache_unpack4<FMT>(w.x, f);
    cache_unpack4<FMT>(w.y, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] *= shrink;
      g[i] *= shrink;
    }
    *dst = make_uint2(cache_pack4<FMT>(f[0], f[1], f[2], f[3]), cache_pack4<FMT>(g[0], g[1], g[2], g[3]));
  }
}

constexpr int READ_THREADS = 256, READ_CHUNKS = 4;  // 8-code chunks per thread

template <int HD, int FMT, int DST>
__global__ void __launch_bounds__(READ_THREADS) cache_read_kernel(const __grid_constant__ CacheReadParams p) {
  constexpr int RC = HD / 8;
  const int b = blockIdx.y / p.Hkv, h = blockIdx.y - b * p.Hkv;
  const CacheSide& S = p.side[blockIdx.z];
  const uint8_t* codes = S.codes + (long long)b * S.sb + (long long)h * S.sh;
  const uint8_t* scale = S.scale + (long long)b * S.scale_sb + (long long)h * S.scale_sh;
  const int live = p.lengths ? p.lengths[b * p.len_step] : p.start + p.n;
  const int ch = threadIdx.x % RC;
  const int r0 = blockIdx.x * (READ_THREADS * READ_CHUNKS / RC) + threadIdx.x / RC;
  uint2 w[READ_CHUNKS];
  int u[READ_CHUNKS];
#pragma unroll
  for (int c = 0; c < READ_CHUNKS; ++c) {
    const int key = p.start + r0 + c * (READ_THREADS / RC);
    w[c] = make_uint2(0, 0);
    u[c] = 0;
    if (key < live && key < p.start + p.n) {
      w[c] = __ldg(reinterpret_cast<const uint2*>(codes + (long long)key * S.ss + ch * 8));
      u[c] = __ldg(scale + (key >> p.log_block));
    }
  }
#pragma unroll
  for (int c = 0; c < READ_CHUNKS; ++c) {
    const int r = r0 + c * (READ_THREADS / RC);
    if (r >= p.n) return;
    const float s = cache_scale(u[c]);
    float f[8], lo[4], hi[4];
    cache_unpack4<FMT>(w[c].x, lo);
    cache_unpack4<FMT>(w[c].y, hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = lo[i] * s;
      f[4 + i] = hi[i] * s;
    }
    const long long off = ((long long)blockIdx.y * p.n + r) * HD + ch * 8;
    if constexpr (DST == CACHE_FP32) {
      float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.dst[blockIdx.z]) + off);
      d[0] = make_float4(f[0], f[1], f[2], f[3]);
      d[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DST == CACHE_BF16) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          o[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.dst[blockIdx.z]) + off) =
          make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <int HD, int FMT, int SRC>
static cudaError_t write_as(const CacheWriteParams& p, int batch, cudaStream_t stream) {
  const int T = 1 << p.log_block;
  // blocks that [pos, pos + n_new) touches; with a device position, the most that any position does
  const int blocks = p.pos_dev ? (p.n_new + 2 * T - 2) / T : (p.pos + p.n_new - 1) / T - p.pos / T + 1;
  cache_write_kernel<HD, FMT, SRC><<<dim3(blocks, batch * p.Hkv, 2), T * HD / 32, 0, stream>>>(p);
  return cudaGetLastError();
}

template <int HD, int FMT, int DST>
static cudaError_t read_as(const CacheReadParams& p, int batch, cudaStream_t stream) {
  constexpr int rows = READ_THREADS * READ_CHUNKS / (HD / 8);  // per CTA
  cache_read_kernel<HD, FMT, DST>
      <<<dim3((p.n + rows - 1) / rows, batch * p.Hkv, 2), READ_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

#define DTA_CACHE_DISPATCH(FN)                                                       \
  template <int HD, int FMT, typename P>                                             \
  static cudaError_t FN##_type(const P& p, int batch, int type, cudaStream_t s) {    \
    return type == CACHE_BF16   ? FN##_as<HD, FMT, CACHE_BF16>(p, batch, s)          \
           : type == CACHE_FP16 ? FN##_as<HD, FMT, CACHE_FP16>(p, batch, s)          \
                                : FN##_as<HD, FMT, CACHE_FP32>(p, batch, s);         \
  }                                                                                  \
  template <typename P>                                                              \
  static cudaError_t FN##_any(const P& p, int batch, int hd, int fmt, int type, cudaStream_t s) { \
    if (hd == 128)                                                                   \
      return fmt == CACHE_E4M3 ? FN##_type<128, CACHE_E4M3>(p, batch, type, s)       \
                               : FN##_type<128, CACHE_INT8>(p, batch, type, s);      \
    return fmt == CACHE_E4M3 ? FN##_type<64, CACHE_E4M3>(p, batch, type, s)          \
                             : FN##_type<64, CACHE_INT8>(p, batch, type, s);         \
  }
DTA_CACHE_DISPATCH(write)
DTA_CACHE_DISPATCH(read)
#undef DTA_CACHE_DISPATCH

cudaError_t launch_cache_write(const CacheWriteParams& p, int batch, int head_dim, int format, int src_type,
                               cudaStream_t stream) {
  return write_any(p, batch, head_dim, format, src_type, stream);
}
cudaError_t launch_cache_read(const CacheReadParams& p, int batch, int head_dim, int format, int dst_type,
                              cudaStream_t stream) {
  return read_any(p, batch, head_dim, format, dst_type, stream);
}

}  // namespace dta
