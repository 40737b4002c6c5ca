// Single-token attention over an 8-bit KV cache (sm_100a).
//
// For one query row per (batch, head), with k_j = K_j 2^(a_j) and v_j = V_j 2^(e_j)
// (codes K, V; block scales 2^a, 2^e):
//   s_j = scaling * log2(e) * 2^(a_j) (q . K_j),   out = sum_j 2^(s_j) 2^(e_j) V_j / sum_j 2^(s_j).
// One pass keeps, per head, the running maxima m = max s_j and r = max (s_j + e_j),
// l = sum 2^(s_j - m) and o = sum 2^(s_j + e_j - r) V_j (fp32); out = o 2^(r - m) / l.
// The value scale enters the exponent, so the weights of o stay in (0, 1] whatever
// the scales are, and are held in fp16 times 2^14 for the tensor cores (11 bits down
// to 2^-28, more than bf16 has); codes convert to fp16 exactly.  Queries are scaled
// per head by a power of two into fp16's range, which is exact down to 2^-29 of the
// head's largest element.
//
// Split-K over the cache: CTA (chunk, batch x KV head) reads its chunk's codes once
// for all G <= 8 query heads of the group; the partials (m, l, r, o) of the chunks
// are merged by a second, dependent launch.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "dta_cache.h"
#include "dta_cache_codes.cuh"
#include "dta_ptx.cuh"

namespace dta {

constexpr int CD_WARPS = 4;
constexpr int CD_THREADS = CD_WARPS * 32;
constexpr float CD_SHIFT = 14.f;  // log2 of the factor that the fp16 weights carry

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of 16-bit values held one row per lane quad.
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 ld_stream16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ int cd_live(const CacheDecodeParams& p, int b) {
  if (!p.n_keys_dev) return p.n_keys;
  return min(max(p.n_keys_dev[b * p.len_step], 0), p.n_keys);
}

// Key range [k0, k1) of launched chunk x of key set `which` with n live keys.
// Dense, and sparse with n <= sink + window: [0, n) in chunks.  Sparse else:
// [0, sink) in n_sink_chunks chunks, then [n - window, n) in the others, whose
// bounds lie on multiples of CACHE_GROUP (the last takes what is left).
__device__ __forceinline__ void cd_range(const CacheDecodeParams& p, const CacheDecodeSet& S, int which, int n, int x,
                                         int& k0, int& k1) {
  if (which == 0 || (long long)n <= (long long)p.sink + p.window) {
    k0 = x * S.chunk;
    k1 = min(k0 + S.chunk, n);
  } else if (x < S.n_sink_chunks) {
    k0 = x * S.chunk;
    k1 = min(k0 + S.chunk, p.sink);
  } else {
    const int w0 = n - p.window, base = w0 & ~(CACHE_GROUP - 1);
    const int i = x - S.n_sink_chunks;
    k0 = max(w0, base + i * S.chunk);
    k1 = x == S.n_launched - 1 ? n : min(base + (i + 1) * S.chunk, n);
  }
  k1 = max(k1, k0);
}

// One group of 16 keys as a warp holds it: K for lane (g, t) = (lane / 4, lane % 4):
// keys g and 8 + g, 16-byte pieces t and t + 4 of the row; V: keys 2t, 2t+1, 2t+8,
// 2t+9, bytes [HD/8 * g, HD/8 * (g + 1)).
template <int HD>
struct Group {
  static constexpr int KP = HD / 64;       // 16-byte pieces per lane and key of K
  static constexpr int VW = HD / 32;       // words per lane and key of V
  uint32_t k[2][KP][4];
  uint32_t v[4][VW];
  int ku, vu;                              // scale bytes
};

template <int HD, int FMT>
__global__ void __launch_bounds__(CD_THREADS) cache_decode_kernel(const __grid_constant__ CacheDecodeParams p, int which) {
  constexpr int KP = HD / 64, VW = HD / 32, NJ = HD / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int b = blockIdx.y / p.Hkv, hk = blockIdx.y - b * p.Hkv;
  const int G = p.G;
  const CacheDecodeSet& S = p.set[which];
  grid_dependents_launch();
  int k0, k1;
  cd_range(p, S, which, cd_live(p, b), blockIdx.x, k0, k1);

  const uint8_t* kc = p.side[0].codes + (long long)b * p.side[0].sb + (long long)hk * p.side[0].sh;
  const uint8_t* vc = p.side[1].codes + (long long)b * p.side[1].sb + (long long)hk * p.side[1].sh;
  const uint8_t* ks = p.side[0].scale + (long long)b * p.side[0].scale_sb + (long long)hk * p.side[0].scale_sh;
  const uint8_t* vs = p.side[1].scale + (long long)b * p.side[1].scale_sb + (long long)hk * p.side[1].scale_sh;

  // Q as the B operand: head g, dims 16 (t + 4c) + 4i + {0, 1} and + {2, 3} for
  // step (c, i), the dims that word i of a lane's piece c holds
  uint32_t qb[KP][4][2];
  float my_scale;
  {
    const bool hv = g < G;
    const __nv_bfloat16* qp = p.q + (long long)b * p.q_sb + (long long)(hk * G + (hv ? g : 0)) * p.q_sh;
    uint4 raw[KP][2];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        raw[c][i] = hv ? reinterpret_cast<const uint4*>(qp + 16 * (t + 4 * c))[i] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max((w[e] << 16) & 0x7fffffffu, w[e] & 0x7fff0000u));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // bring the largest magnitude to [2^14, 2^15); a row with a non-finite element is NaN throughout
    const int e = (int)(top >> 23);
    const int up = e == 255 ? 0 : min(max(141 - e, -126), 126);
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    my_scale = e == 255 ? __uint_as_float(0x7fc00000u) : p.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2)
          qb[c][2 * i + (e2 >> 1)][e2 & 1] =
              pack_f16x2(__uint_as_float(w[e2] << 16) * f, __uint_as_float(w[e2] & 0xffff0000u) * f);
      }
  }
  // score factors of this lane's columns, heads 2t and 2t + 1
  float sl[2];
  sl[0] = __shfl_sync(0xffffffffu, my_scale, 8 * t);
  sl[1] = __shfl_sync(0xffffffffu, my_scale, 8 * t + 4);

  float m[2] = {-INFINITY, -INFINITY}, r[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  auto load = [&](int base, Group<HD>& x) {
    const bool whole = base >= k0 && base + CACHE_GROUP <= k1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = base + 8 * e + g;
      const bool ok = whole || (key >= k0 && key < k1);
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        const uint4 w = ok ? ld_stream16(kc + (long long)key * p.side[0].ss + 16 * (t + 4 * c)) : make_uint4(0, 0, 0, 0);
        x.k[e][c][0] = w.x; x.k[e][c][1] = w.y; x.k[e][c][2] = w.z; x.k[e][c][3] = w.w;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = base + 8 * (e >> 1) + 2 * t + (e & 1);
      const bool ok = whole || (key >= k0 && key < k1);  // (a masked value must not be NaN: 0 * NaN)
      const uint8_t* src = vc + (long long)key * p.side[1].ss + 4 * VW * g;
      if constexpr (VW == 4) {
        const uint4 w = ok ? ld_stream16(src) : make_uint4(0, 0, 0, 0);
        x.v[e][0] = w.x; x.v[e][1] = w.y; x.v[e][2] = w.z; x.v[e][3] = w.w;
      } else {
        const uint2 w = ok ? *reinterpret_cast<const uint2*>(src) : make_uint2(0, 0);
        x.v[e][0] = w.x; x.v[e][1] = w.y;
      }
    }
    const int blk = base >> p.log_block;
    x.ku = ks[blk];
    x.vu = vs[blk];
  };

  auto step = [&](int base, const Group<HD>& x) {
    // S^T (keys x heads) = K Q^T
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w0 = cache_bias<FMT>(x.k[0][c][i]), w1 = cache_bias<FMT>(x.k[1][c][i]);
        mma_f16(s, cache_half2<FMT, 0>(w0), cache_half2<FMT, 0>(w1), cache_half2<FMT, 1>(w0), cache_half2<FMT, 1>(w1),
                qb[c][i][0], qb[c][i][1]);
      }
    const float kf = cache_scale(x.ku);
    const float ve = x.vu == 255 ? __uint_as_float(0x7fc00000u) : (float)(x.vu - 127);
    const int key = base + g;
    const bool ok0 = key >= k0 && key < k1, ok1 = key + 8 >= k0 && key + 8 < k1;
    float pw[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float f = sl[h] * kf;
      const float s0 = ok0 ? s[h] * f : -INFINITY, s1 = ok1 ? s[2 + h] * f : -INFINITY;
      float mx = fmaxf(s0, s1);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float mn = fmaxf(m[h], mx), rn = fmaxf(r[h], mx + ve);
      const float mu = mn == -INFINITY ? 0.f : mn, ru = rn == -INFINITY ? 0.f : rn;
      const float am = fast_exp2(m[h] - mu), ar = fast_exp2(r[h] - ru);
      m[h] = mn;
      r[h] = rn;
      l[h] = l[h] * am + fast_exp2(s0 - mu) + fast_exp2(s1 - mu);
      const float off = ve - ru + CD_SHIFT;
      pw[h] = fast_exp2(s0 + off);
      pw[2 + h] = fast_exp2(s1 + off);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        o[j][h] *= ar;
        o[j][2 + h] *= ar;
      }
    }
    // P^T as the B operand: keys 2t, 2t+1 (and 8 more), head g
    const uint32_t b0 = movmatrix_t(pack_f16x2(pw[0], pw[1]));
    const uint32_t b1 = movmatrix_t(pack_f16x2(pw[2], pw[3]));
    // O^T (dims x heads) += V^T P^T; rows g and 8 + g of tile j are dims HD/8 g + 2j, + 1
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      const uint32_t wa = cache_bias<FMT>(x.v[0][i]), wb = cache_bias<FMT>(x.v[1][i]);
      const uint32_t wc = cache_bias<FMT>(x.v[2][i]), wd = cache_bias<FMT>(x.v[3][i]);
      const uint32_t ab = __byte_perm(wa, wb, 0x5140), AB = __byte_perm(wa, wb, 0x7362);
      const uint32_t cd = __byte_perm(wc, wd, 0x5140), CD = __byte_perm(wc, wd, 0x7362);
      mma_f16(o[2 * i], cache_half2<FMT, 0>(ab), cache_half2<FMT, 1>(ab), cache_half2<FMT, 0>(cd),
              cache_half2<FMT, 1>(cd), b0, b1);
      mma_f16(o[2 * i + 1], cache_half2<FMT, 0>(AB), cache_half2<FMT, 1>(AB), cache_half2<FMT, 0>(CD),
              cache_half2<FMT, 1>(CD), b0, b1);
    }
  };

  const int first = (k0 & ~(CACHE_GROUP - 1)) + warp * CACHE_GROUP;
  constexpr int STEP = CD_WARPS * CACHE_GROUP;
  Group<HD> x;
  if (first < k1) load(first, x);
  for (int base = first; base < k1; base += STEP) {
    Group<HD> nx;
    if (base + STEP < k1) load(base + STEP, nx);
    step(base, x);
    x = nx;
  }

  // merge the warps through shared memory
  __shared__ float red_o[CD_WARPS][8][HD];
  __shared__ float red_s[CD_WARPS][3][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
    if (g == 0) {
      red_s[warp][0][2 * t + h] = m[h];
      red_s[warp][1][2 * t + h] = l[h];
      red_s[warp][2][2 * t + h] = r[h];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      red_o[warp][2 * t + h][HD / 8 * g + 2 * j] = o[j][h];
      red_o[warp][2 * t + h][HD / 8 * g + 2 * j + 1] = o[j][2 + h];
    }
  }
  __syncthreads();
  float* part0 = S.partials + ((long long)(b * p.H + hk * G) * S.n_launched + blockIdx.x) * (4 + HD);
  for (int idx = threadIdx.x; idx < G * HD; idx += CD_THREADS) {
    const int h = idx / HD, d = idx - h * HD;
    float M = -INFINITY, R = -INFINITY;
#pragma unroll
    for (int w = 0; w < CD_WARPS; ++w) {
      M = fmaxf(M, red_s[w][0][h]);
      R = fmaxf(R, red_s[w][2][h]);
    }
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < CD_WARPS; ++w) {
      if (red_s[w][1][h] == 0.f) continue;  // no key of this warp counts
      L += red_s[w][1][h] * fast_exp2(red_s[w][0][h] - M);
      O += red_o[w][h][d] * fast_exp2(red_s[w][2][h] - R);
    }
    float* part = part0 + (long long)h * S.n_launched * (4 + HD);
    part[4 + d] = O;
    if (d == 0) {
      part[0] = M;
      part[1] = L;
      part[2] = R;
    }
  }
}

// Merge of a key set's partials: grid (B * H), one thread per head dim.
template <int HD>
__global__ void cache_merge_kernel(const __grid_constant__ CacheDecodeParams p) {
  const int bh = blockIdx.x, d = threadIdx.x;
  grid_dependency_wait();
  for (int which = 0; which < 2; ++which) {
    if (!p.out[which]) continue;
    const CacheDecodeSet& S = p.set[which];
    const float* base = S.partials + (long long)bh * S.n_launched * (4 + HD);
    float M = -INFINITY, R = -INFINITY, L = 0.f, O = 0.f;
    for (int x = 0; x < S.n_launched; ++x) {
      const float* part = base + (long long)x * (4 + HD);
      const float m = part[0], l = part[1], r = part[2], o = part[4 + d];
      if (l == 0.f) continue;
      const float mn = fmaxf(M, m), rn = fmaxf(R, r);
      L = L * fast_exp2(M - mn) + l * fast_exp2(m - mn);
      O = O * fast_exp2(R - rn) + o * fast_exp2(r - rn);
      M = mn;
      R = rn;
    }
    const float v = L == 0.f ? 0.f : (O * 0x1p-14f) * exp2f(R - M) / L;
    p.out[which][(long long)bh * HD + d] = __float2bfloat16_rn(v);
  }
}

template <int HD, int FMT>
static cudaError_t decode_as(const CacheDecodeParams& p, cudaStream_t stream) {
  for (int which = 0; which < 2; ++which)
    if (p.out[which])
      cache_decode_kernel<HD, FMT><<<dim3(p.set[which].n_launched, p.B * p.Hkv), CD_THREADS, 0, stream>>>(p, which);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cache_merge_kernel<HD><<<p.B * p.H, HD, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_cache_decode(const CacheDecodeParams& p, int head_dim, int format, cudaStream_t stream) {
  if (head_dim == 128)
    return format == CACHE_E4M3 ? decode_as<128, CACHE_E4M3>(p, stream) : decode_as<128, CACHE_INT8>(p, stream);
  return format == CACHE_E4M3 ? decode_as<64, CACHE_E4M3>(p, stream) : decode_as<64, CACHE_INT8>(p, stream);
}

}  // namespace dta
