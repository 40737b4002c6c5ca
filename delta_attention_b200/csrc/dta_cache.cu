// Writing an 8-bit KV cache and reading it back (sm_100a).
//
// Write: a scale block of one head of K or V belongs to one group of threads.
// It fetches the block's new rows once, reduces their largest finite magnitude,
// and stores the codes; a block that already holds earlier tokens keeps the
// larger of its own and the new scale, and where that raises the scale the
// group rounds the earlier codes to it.  Nothing is shared between blocks.
// Read: codes times their block's scale, rounded once.
// Both are streams, bound by the memory traffic once the conversions are cheap
// enough.  131072 tokens x 8 heads x 128 dims of K and V, bf16 to e4m3: 117 us, 6.9
// TB/s of values read and codes written; with one conversion and one comparison per
// element the ALUs bound it (147 us).  65536 x 8 x 128 read back to bf16: 61.7 us,
// 6.5 TB/s; one 8-byte load per thread instead of four in flight took 90.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "dta_cache.h"
#include "dta_cache_codes.cuh"
#include "dta_ptx.cuh"

namespace dta {

// Sixteen bytes of a source row: 8 elements, or 4 of fp32.  `top` folds their
// magnitudes into a running maximum (NaN stays), `bits` gives the bits of that
// maximum as fp32, `get` the elements as pairs of fp32.
template <int SRC>
struct Piece;
template <>
struct Piece<CACHE_BF16> {
  static constexpr int N = 8;
  uint4 r;
  static __device__ __forceinline__ uint32_t max_abs(uint32_t m, uint32_t x) {
    asm("{\n\t.reg .b32 a;\n\tabs.bf16x2 a, %1;\n\tmax.NaN.bf16x2 %0, %0, a;\n\t}" : "+r"(m) : "r"(x));
    return m;
  }
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = max_abs(max_abs(max_abs(max_abs(m, r.x), r.y), r.z), r.w);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return max(m & 0x7fffu, (m >> 16) & 0x7fffu) << 16; }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <>
struct Piece<CACHE_FP16> {
  static constexpr int N = 8;
  uint4 r;
  static __device__ __forceinline__ uint32_t max_abs(uint32_t m, uint32_t x) {
    asm("{\n\t.reg .b32 a;\n\tabs.f16x2 a, %1;\n\tmax.NaN.f16x2 %0, %0, a;\n\t}" : "+r"(m) : "r"(x));
    return m;
  }
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = max_abs(max_abs(max_abs(max_abs(m, r.x), r.y), r.z), r.w);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0x7fffu, (m >> 16) & 0x7fffu))));
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
};
template <>
struct Piece<CACHE_FP32> {
  static constexpr int N = 4;
  uint4 r;
  __device__ __forceinline__ void top(uint32_t& m) const {  // (as integers: infinity and NaN lie above the finite)
    m = max(max(m, r.x & 0x7fffffffu), r.y & 0x7fffffffu);
    m = max(max(m, r.z & 0x7fffffffu), r.w & 0x7fffffffu);
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t m) { return m; }
  __device__ __forceinline__ void get(float2 (&f)[2]) const {
    f[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    f[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
};

__device__ __forceinline__ bool finite32(float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; }

// The codes of one piece to `dst`.  `clean`: every value is finite.  Else a
// non-finite value becomes NaN (e4m3, which has no infinity); an int8 block that
// holds one reads as NaN by its scale and gets zeros.
template <int FMT, int SRC>
__device__ __forceinline__ void store_codes(const Piece<SRC>& x, float inv, bool clean, uint8_t* dst) {
  constexpr int N = Piece<SRC>::N;
  float2 f[N / 2];
  x.get(f);
  uint32_t w[N / 4];
  if (clean) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = cache_pack4<FMT>(f[2 * i], f[2 * i + 1], inv);
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float v[4] = {f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y};
      float g[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = finite32(v[e]) ? v[e] : 0.f;
      w[i] = FMT == CACHE_INT8 ? 0u : cache_pack4<FMT>(make_float2(g[0], g[1]), make_float2(g[2], g[3]), inv);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (FMT == CACHE_E4M3 && !finite32(v[e])) w[i] |= 0x7fu << (8 * e);
    }
  }
  if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

constexpr int WRITE_ELEMS = 64;     // elements per thread
constexpr int WRITE_THREADS = 128;  // at least; a block of 128 x 128 takes 256

// Threads [0, group), [group, 2 group), ... of a CTA each get their own largest
// value.  `red` holds a word per warp and is free again after the next barrier.
__device__ __forceinline__ uint32_t group_max(uint32_t v, int group, uint32_t* red) {
#pragma unroll
  for (int d = 1; d < 16; d *= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  if (group >= 32) v = max(v, __shfl_xor_sync(0xffffffffu, v, 16));
  if (group <= 32) return v;
  const int warp = threadIdx.x >> 5, n = group >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  for (int w = 0; w < n; ++w) v = max(v, red[(warp & ~(n - 1)) + w]);
  return v;
}

// Each group of T * HD / 64 threads quantises one scale block; a CTA has 128
// threads' worth of consecutive blocks.  The rows are staged in shared memory by
// asynchronous copies, each thread's share its own (so no barrier comes between the
// copies and the reads), which keeps 16 KB per CTA in flight at few registers.  A
// thread's pieces lie in one column, T * N / 64 rows apart.
template <int HD, int FMT, int SRC>
__global__ void __launch_bounds__(256) cache_write_kernel(const __grid_constant__ CacheWriteParams p) {
  constexpr int N = Piece<SRC>::N, RC = HD / N, PIECES = WRITE_ELEMS / N, ES = 16 / N;
  extern __shared__ __align__(16) uint4 staged[];
  __shared__ uint32_t red[2][8];
  // heads vary fastest: CTAs that run together read neighbouring heads' rows of the
  // same tokens, which lie next to each other in a projection's output
  const int b = blockIdx.y, slab = blockIdx.x / p.Hkv, h = blockIdx.x - slab * p.Hkv;
  const int side = blockIdx.z;
  const CacheSide& S = p.side[side];
  grid_dependency_wait();
  grid_dependents_launch();
  // [first, end): the positions that this call writes in sequence b
  const int first = p.pos_dev ? p.pos_dev[b * p.pos_step] : p.pos;
  const int len = p.lengths ? p.lengths[b * p.len_step] : p.n_new;
  if (first < 0 || first > p.capacity || len < 0 || len > p.n_new || len > p.capacity - first) {
    // a device position or length outside the cache: nothing of this sequence is written
    if (threadIdx.x == 0 && blockIdx.x == 0 && p.error_word) atomicCAS(p.error_word, 0, (int)KERR_BAD_ROW);
    return;
  }
  const int end = first + len;
  const int log_group = p.log_block + (HD == 128 ? 1 : 0), group = 1 << log_group;
  const int tg = threadIdx.x & (group - 1);
  const int per_cta = blockDim.x >> log_group;
  const int blk0 = (first >> p.log_block) + slab * per_cta;
  // the whole CTA is past the end (compared in blocks: their positions may pass 2^31)
  if (len == 0 || blk0 > (end - 1) >> p.log_block) return;
  const int blk = blk0 + (threadIdx.x >> log_group);
  const int lo = blk << p.log_block;
  const int T = 1 << p.log_block, dr = group / RC;  // rows of a block, rows between a thread's pieces
  const int t0 = lo + tg / RC, col = tg % RC;
  const bool whole = lo >= first && lo + T <= end;

  const long long src_ss = p.src_ss[side] * ES;
  const char* src = reinterpret_cast<const char*>(p.src[side]) +
                    ((long long)b * p.src_sb[side] + (long long)h * p.src_sh[side]) * ES + col * 16;
  const uint32_t slot = smem_u32(staged + threadIdx.x), slots = blockDim.x * 16;
  if (whole) {
    const char* at = src + (long long)(t0 - first) * src_ss;
#pragma unroll
    for (int c = 0; c < PIECES; ++c, at += dr * src_ss) cp_async_16(slot + c * slots, at, 16u);
  } else {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const int t = t0 + c * dr;
      const bool fresh = t >= first && t < end;  // other rows are zeros
      cp_async_16(slot + c * slots, src + (fresh ? (long long)(t - first) * src_ss : 0), fresh ? 16u : 0u);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  const bool held = lo < first;  // the block holds tokens before this call's first
  uint8_t* codes = S.codes + (long long)b * S.sb + (long long)h * S.sh + col * N;
  uint8_t* scale = S.scale + (long long)b * S.scale_sb + (long long)h * S.scale_sh + blk;
  const int u_old = held ? *scale : 0;
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  const uint4* mine = staged + threadIdx.x;
  Piece<SRC> x;
  uint32_t amax = 0;
#pragma unroll
  for (int c = 0; c < PIECES; ++c) {
    x.r = mine[c * blockDim.x];
    x.top(amax);
  }
  amax = group_max(Piece<SRC>::bits(amax), group, red[0]);
  const bool clean = amax < 0x7f800000u;
  if (FMT == CACHE_E4M3 && __syncthreads_or(!clean)) {  // the scale goes by the finite values
    float top = 0.f;
    for (int c = 0; c < PIECES; ++c) {
      float2 f[N / 2];
      x.r = mine[c * blockDim.x];
      x.get(f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (finite32(f[i].x)) top = fmaxf(top, fabsf(f[i].x));
        if (finite32(f[i].y)) top = fmaxf(top, fabsf(f[i].y));
      }
    }
    amax = group_max(__float_as_uint(top), group, red[1]);
  } else {
    __syncthreads();  // every thread has read its block's old scale
  }
  if (lo >= end) return;
  const int u = max(amax >= 0x7f800000u ? 255 : cache_need<FMT>(__uint_as_float(amax)), u_old);
  if (tg == 0) *scale = (uint8_t)u;
  const float inv = u == 255 ? 0.f : cache_inv_scale(u);
  uint8_t* dst = codes + (long long)t0 * S.ss;
  if (whole && clean) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c, dst += dr * S.ss) {
      x.r = mine[c * blockDim.x];
      store_codes<FMT, SRC>(x, inv, true, dst);
    }
    return;
  }
  for (int c = 0; c < PIECES; ++c, dst += dr * S.ss) {
    const int t = t0 + c * dr;
    if (t < first || t >= end) continue;
    x.r = mine[c * blockDim.x];
    store_codes<FMT, SRC>(x, inv, clean, dst);
  }
  if (!held || u == u_old) return;
  // the scale rose: the block's earlier codes are rounded to it
  const float shrink = u - u_old > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (u - u_old)) << 23);
  dst = codes + (long long)t0 * S.ss;
  for (int t = t0; t < first; t += dr, dst += dr * S.ss) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      uint32_t* w = reinterpret_cast<uint32_t*>(dst) + i;
      float f[4];
      cache_unpack4<FMT>(*w, f);
      // (an e4m3 NaN stays one: NaN times anything converts to NaN)
      *w = cache_pack4<FMT>(make_float2(f[0], f[1]), make_float2(f[2], f[3]), shrink);
    }
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
  grid_dependency_wait();
  grid_dependents_launch();
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
      w[c] = *reinterpret_cast<const uint2*>(codes + (long long)key * S.ss + ch * 8);
      u[c] = scale[key >> p.log_block];
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

// Launches as a programmatic dependent: the kernel's CTAs may come up while the last
// kernel on the stream drains, and wait for it before they touch memory.
template <typename P>
static cudaError_t launch_dependent(void (*kernel)(P), dim3 grid, int threads, int smem, cudaStream_t stream,
                                    const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int HD, int FMT, int SRC>
static cudaError_t write_as(const CacheWriteParams& p, int batch, cudaStream_t stream) {
  const int T = 1 << p.log_block, group = T * HD / 64;
  const int threads = group > WRITE_THREADS ? group : WRITE_THREADS, per_cta = threads / group;
  // blocks that [pos, pos + n_new) touches; with a device position, the most that any position does
  const int blocks = p.pos_dev ? (p.n_new + 2 * T - 2) / T : (p.pos + p.n_new - 1) / T - p.pos / T + 1;
  const int smem = threads * WRITE_ELEMS * (16 / Piece<SRC>::N);  // 16 to 64 KB
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(cache_write_kernel<HD, FMT, SRC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid((unsigned)((blocks + per_cta - 1) / per_cta) * p.Hkv, batch, 2);
  return launch_dependent(cache_write_kernel<HD, FMT, SRC>, grid, threads, smem, stream, p);
}

template <int HD, int FMT, int DST>
static cudaError_t read_as(const CacheReadParams& p, int batch, cudaStream_t stream) {
  constexpr int rows = READ_THREADS * READ_CHUNKS / (HD / 8);  // per CTA
  const dim3 grid((p.n + rows - 1) / rows, batch * p.Hkv, 2);
  return launch_dependent(cache_read_kernel<HD, FMT, DST>, grid, READ_THREADS, 0, stream, p);
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
