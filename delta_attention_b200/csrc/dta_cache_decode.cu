// Single-token attention over an 8-bit KV cache (sm_100a).
//
// For one query row per (batch, head), with k_j = K_j 2^(a_j) and v_j = V_j 2^(e_j)
// (codes K, V; block scales 2^a, 2^e):
//   s_j = scaling * log2(e) * 2^(a_j) (q . K_j),   out = sum_j 2^(s_j) 2^(e_j) V_j / sum_j 2^(s_j).
// One pass keeps, per head, the running maxima m = max s_j and r = max (s_j + e_j),
// l = sum 2^(s_j - m) and o = sum 2^(s_j + e_j - r) V_j (fp32); out = o 2^(r - m) / l.
// The value scale enters the exponent, so the weights of o stay in (0, 1] whatever
// the scales are, and are held in fp16 times 2^14 for the tensor cores (11 bits down
// to 2^-28, more than bf16 has); value codes are exact in fp16.
//
// The scores' operands.  e4m3: codes and queries in fp16, the queries scaled per head
// by a power of two so that the largest element lies in [2^14, 2^15) (exact down to
// 2^-29 of it); products and sums in fp32.  (With the 8-bit mma.sync of this type the
// kernel executed 25% more instructions.)  int8: codes as they
// are, the queries times a power of two per head that brings the largest element to
// [2^22, 2^23), as 24-bit integers in three 8-bit parts (bf16's bits are all kept down to
// 2^-15 of the largest element, smaller ones are off by at most 2^-23 of it); products and
// sums in integers.  With two parts (2^-16 of it) a query with one channel 200 times the
// others was off by more than the output's rounding to bf16.  The third costs 4% where calls
// follow one another for long (4 x 65536 keys, both rows, d 128: 93.5 us for 90.0; dense, 4 x
// 131072, d 64: 102.7 for 99.1), nothing at d 128 in short runs (87.9 for 89.1); four parts,
// two to a product where a group has 4 heads at most, took as long.  With codes converted
// to fp16 the first of these took 102 us where two parts took 92.
//
// Split-K over the cache: CTA (chunk, batch x KV head) reads its chunk's codes once
// for all G <= 8 query heads of the group; the partials (m, l, r, o) of the chunks
// are merged within a thread-block cluster or by a second, dependent launch.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "dta_cache.h"
#include "dta_cache_codes.cuh"
#include "dta_ptx.cuh"

namespace dta {

constexpr int CD_WARPS = 4;
constexpr int CD_THREADS = CD_WARPS * 32;
template <int HD>
constexpr int CD_KEYS = cache_step(HD) / CD_WARPS;  // keys per step of a warp: 4 KB of K and of V
constexpr int CD_STAGES = 3;  // steps in flight per warp
constexpr float CD_SHIFT = 14.f;  // log2 of the factor that the fp16 weights carry

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A signed; B signed, or with `US` unsigned.
template <bool US>
__device__ __forceinline__ void mma_int8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (US)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
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

// Live keys of sequence b.
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

// Merging partials (m, l, r, o) of chunks by the log-sum-exp rule.  The lanes of a
// warp hold the headers (32 per array element); every lane ends up with the total.
constexpr int MG_ROWS = 4, MG_LOADS = 16;
template <int HEADS>
struct MergeState {
  float M, R, L;
  __device__ __forceinline__ void start() {
    M = R = -INFINITY;
    L = 0.f;
  }
  // Takes more chunks: wo their factors on o (-1 for a chunk without keys, whose o was
  // never written); returns the factor that brings the o of earlier chunks to the new maximum.
  __device__ __forceinline__ float weigh(const float (&m)[HEADS], const float (&l)[HEADS], const float (&r)[HEADS],
                                         float (&wo)[HEADS]) {
    float mt = M, rt = R;
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
      mt = fmaxf(mt, m[k]);
      rt = fmaxf(rt, r[k]);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) {
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
      rt = fmaxf(rt, __shfl_xor_sync(0xffffffffu, rt, x));
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
      sum += l[k] == 0.f ? 0.f : l[k] * fast_exp2(m[k] - mt);
      wo[k] = l[k] == 0.f ? -1.f : fast_exp2(r[k] - rt);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    L = (M == mt ? L : L * fast_exp2(M - mt)) + sum;
    const float f = R == rt ? 1.f : fast_exp2(R - rt);
    M = mt;
    R = rt;
    return f;
  }
  __device__ __forceinline__ __nv_bfloat16 finish(float o) const {
    return __float2bfloat16_rn(L == 0.f ? 0.f : (o * 0x1p-14f) * exp2f(R - M) / L);
  }
};
// (A factor of 0 is applied: a chunk far below the maximum, or with no finite r, may hold a NaN, which stays.)
__device__ __forceinline__ void merge_add(float& acc, float o, float w) { acc = w < 0.f ? acc : fmaf(o, w, acc); }
constexpr int CD_CLUSTER_MAX = 16;  // CTAs of a cluster (above 8: non-portable sizes, used where they fit)

// Shared-memory ring of one warp: CD_STAGES stages of CD_KEYS keys, each K rows
// then V rows of HD bytes.  The 16-byte pieces of row r are permuted by r, so
// that the fragment reads below are free of bank conflicts (HD = 128; at 64 the
// reads of V take two passes).
template <int HD>
__device__ __forceinline__ int cd_swizzle(int row, int piece) {
  return HD == 128 ? piece ^ (row & 7) : piece ^ (row & 2);
}
template <int HD>
__host__ __device__ constexpr int cd_smem() {
  return CD_WARPS * CD_STAGES * 2 * CD_KEYS<HD> * HD;
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t (&w)[2]) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// Partial kernel: CD_WARPS warps, each with a ring and a state of its own; warp w
// takes the chunk's keys in steps of CD_KEYS, every CD_WARPS-th step.  With
// (g, t) = (lane / 4, lane % 4) a step is, for each group of 16 keys,
//   S^T (16 keys x 8 heads) = K Q^T   A rows g and 8 + g = those keys; lane t holds
//                                     pieces KP t + c of a row; a word of four codes is a
//                                     lane's part of one m16n8k16 step (e4m3), two words
//                                     of one m16n8k32 step (int8)
//   O^T (dims x 8 heads) += V^T P^T   lane (g, t) holds bytes [HD/8 g, HD/8 (g + 1)) of
//                                     keys 2t, 2t+1, 2t+8, 2t+9: rows g and 8 + g of
//                                     tile j are dims HD/8 g + 2j and + 1
// so that codes go from shared memory into fragments without any exchange; only
// the weights are transposed (movmatrix).
//
// The grid's y covers the dense set's chunks and then the sparse set's, so a call
// that wants both rows is one launch, whose short sparse chunks start last (and find
// the sink and window in L2); its x the (batch, KV head) pairs.  CLU: the y extent is
// one thread-block cluster per pair, and the cluster merges its chunks' partials through
// distributed shared memory; else they go to global memory and cache_merge_kernel
// merges them.  Both merge in one order, so calls with the same plan give the same row bit
// for bit whichever way they merge.
//
// Why this shape.  At 8 bits a key costs half the memory time that it costs at 16, so
// the instructions per key decide nearly as much as the memory does: 252 for 16 keys
// (e4m3, 64 of them convert V and K; int8 368), and the kernel without its copies takes 0.6 of
// the time of one without its products.  Hence rings per warp (no barrier in the loop),
// 32 keys a step, maxima that move by vote, and two CTAs of 4 warps per SM with 16 KB per
// warp on the way; 12 warps with 8 KB each, 16-key steps, and K and V in rings of their own
// were slower.  131072 keys, 8 KV heads x 4 queries, d 128, e4m3: 45.9 us with the merge,
// 5.8 TB/s (the copies alone take 43.4); 4 x 65536: 82 us, 6.5 TB/s.
template <int HD, int FMT, bool CLU>
__global__ void __launch_bounds__(CD_THREADS) cache_decode_kernel(const __grid_constant__ CacheDecodeParams p) {
  constexpr int KEYS = CD_KEYS<HD>, NG = KEYS / CACHE_GROUP;
  constexpr int KP = HD / 64, VW = HD / 32, NJ = HD / 16;
  extern __shared__ __align__(128) uint8_t cd_ring[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int b = blockIdx.x / p.Hkv, hk = blockIdx.x - b * p.Hkv;
  const int G = p.G;
  const int n_dense = p.out[0] ? p.set[0].n_launched : 0;
  const int which = (int)blockIdx.y < n_dense ? 0 : 1, chunk = blockIdx.y - (which ? n_dense : 0);
  const CacheDecodeSet& S = p.set[which];
  grid_dependency_wait();    // launched as a programmatic dependent of whatever ran before
  grid_dependents_launch();  // (the merge launch, which waits for this grid in turn)
  int k0, k1;
  cd_range(p, S, which, cd_live(p, b), chunk, k0, k1);

  if (!CLU && k0 >= k1) {  // no keys: an empty partial (its o is not read)
    if (threadIdx.x < G)
      *reinterpret_cast<float4*>(S.partials + ((long long)(b * p.H + hk * G + threadIdx.x) * S.n_launched + chunk) *
                                                  (4 + HD)) = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    return;
  }

  const uint8_t* kc = p.side[0].codes + (long long)b * p.side[0].sb + (long long)hk * p.side[0].sh;
  const uint8_t* vc = p.side[1].codes + (long long)b * p.side[1].sb + (long long)hk * p.side[1].sh;
  const uint8_t* ks = p.side[0].scale + (long long)b * p.side[0].scale_sb + (long long)hk * p.side[0].scale_sh;
  const uint8_t* vs = p.side[1].scale + (long long)b * p.side[1].scale_sb + (long long)hk * p.side[1].scale_sh;
  const long long kss = p.side[0].ss, vss = p.side[1].ss;

  // ---- copies: lane -> piece lane % PC of rows lane / PC, + 32 / PC, ... ----
  constexpr int PC = HD / 16, RL = 32 / PC;  // pieces per row, rows per pass
  constexpr int STAGE = 2 * KEYS * HD;
  const uint32_t ring = smem_u32(cd_ring) + warp * CD_STAGES * STAGE;
  const int cr = lane / PC, cp = lane % PC;
  const int a0 = (k0 & ~(CACHE_GROUP - 1)) + warp * KEYS;
  constexpr int STRIDE = CD_WARPS * KEYS;
  const int steps = k1 > a0 ? (k1 - a0 + STRIDE - 1) / STRIDE : 0;
  // shared-memory offsets of this lane's pieces of its first and second row (the
  // permutation repeats after two passes)
  const uint32_t c0 = cr * HD + (cd_swizzle<HD>(cr, cp) << 4);
  const uint32_t c1 = (cr + RL) * HD + (cd_swizzle<HD>(cr + RL, cp) << 4);
  const bool packed = kss == HD && vss == HD;
  auto issue = [&](int step, int slot) {
    const int base = a0 + step * STRIDE;
    const uint32_t dst = ring + slot * STAGE;
    const uint8_t* ksrc = kc + (long long)(base + cr) * kss + cp * 16;
    const uint8_t* vsrc = vc + (long long)(base + cr) * vss + cp * 16;
    if (base >= k0 && base + KEYS <= k1) {
      if (packed) {  // rows follow one another: every offset is a constant
#pragma unroll
        for (int i = 0; i < KEYS / RL; ++i)
          cp_async_16(dst + (i & 1 ? c1 : c0) + (i >> 1) * 2 * RL * HD, ksrc + i * RL * HD, 16u);
#pragma unroll
        for (int i = 0; i < KEYS / RL; ++i)
          cp_async_16(dst + (i & 1 ? c1 : c0) + (i >> 1) * 2 * RL * HD + KEYS * HD, vsrc + i * RL * HD, 16u);
      } else {
#pragma unroll
        for (int i = 0; i < KEYS / RL; ++i) {
          const uint32_t off = dst + (i & 1 ? c1 : c0) + (i >> 1) * 2 * RL * HD;
          cp_async_16(off, ksrc + i * RL * kss, 16u);
          cp_async_16(off + KEYS * HD, vsrc + i * RL * vss, 16u);
        }
      }
    } else {
      // rows outside the chunk are filled with zeros (a masked value must not be NaN: 0 * NaN)
#pragma unroll
      for (int i = 0; i < KEYS / RL; ++i) {
        const int key = base + cr + i * RL;
        const bool ok = key >= k0 && key < k1;
        const uint32_t off = dst + (i & 1 ? c1 : c0) + (i >> 1) * 2 * RL * HD;
        cp_async_16(off, ok ? ksrc + i * RL * kss : kc + (long long)k0 * kss, ok ? 16u : 0u);
        cp_async_16(off + KEYS * HD, ok ? vsrc + i * RL * vss : vc + (long long)k0 * vss, ok ? 16u : 0u);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < CD_STAGES - 1; ++s) {
    if (s < steps) issue(s, s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // ---- Q as the B operand: entry (c, i) holds head g's dims 16 (KP t + c) + 4 i + {0 .. 3}: as two
  // fp16 pairs (e4m3), or their high, middle and low bytes (int8) ----
  constexpr int QW = FMT == CACHE_E4M3 ? 2 : 3;
  uint32_t qb[KP][4][QW];
  float my_scale;
  {
    const bool hv = g < G;
    const __nv_bfloat16* qp = p.q + (long long)b * p.q_sb + (long long)(hk * G + (hv ? g : 0)) * p.q_sh;
    uint32_t w[KP][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 x = hv ? reinterpret_cast<const uint4*>(qp + 16 * (KP * t + c))[i] : make_uint4(0, 0, 0, 0);
        w[c][4 * i] = x.x; w[c][4 * i + 1] = x.y; w[c][4 * i + 2] = x.z; w[c][4 * i + 3] = x.w;
      }
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, max((w[c][e] << 16) & 0x7fffffffu, w[c][e] & 0x7fff0000u));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the head's power of two: its largest element goes to [2^14, 2^15) (e4m3) or [2^22, 2^23) (int8;
    // heads below 2^-104 keep fewer bits)
    const int up = min(max((FMT == CACHE_E4M3 ? 141 : 149) - (int)(top >> 23), -126), 126);
    float f = __uint_as_float((uint32_t)(127 + up) << 23);
    my_scale = p.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
    // a row with a non-finite element is NaN throughout
    if (top >= 0x7f800000u) {
      f = 0.f;
      my_scale = __uint_as_float(0x7fc00000u);
    }
#pragma unroll
    for (int c = 0; c < KP; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          d[2 * e] = __uint_as_float(w[c][2 * i + e] << 16) * f;
          d[2 * e + 1] = __uint_as_float(w[c][2 * i + e] & 0xffff0000u) * f;
        }
        if constexpr (FMT == CACHE_E4M3) {
          qb[c][i][0] = pack_f16x2(d[0], d[1]);
          qb[c][i][1] = pack_f16x2(d[2], d[3]);
        } else {
          qb[c][i][0] = qb[c][i][1] = qb[c][i][2] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = (uint32_t)__float2int_rn(d[e]);  // |x| < 2^23: 2^16 (signed byte) + 2^8 byte + byte
            qb[c][i][0] |= (x >> 16 & 255) << (8 * e);
            qb[c][i][1] |= (x >> 8 & 255) << (8 * e);
            qb[c][i][2] |= (x & 255) << (8 * e);
          }
        }
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

  // fragment read offsets within a stage (the pieces' permutation depends on the lane alone)
  uint32_t ka[KP], va[2];
#pragma unroll
  for (int c = 0; c < KP; ++c) ka[c] = g * HD + (cd_swizzle<HD>(g, KP * t + c) << 4);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    va[e] = KEYS * HD + (2 * t + e) * HD + (cd_swizzle<HD>(2 * t + e, HD == 128 ? g : g >> 1) << 4) +
            (HD == 128 ? 0 : 8 * (g & 1));

  int slot = 0;
  for (int step = 0; step < steps; ++step) {
    const int base = a0 + step * STRIDE;
    const uint32_t st = ring + slot * STAGE;
    // this step's scale bytes (a group behind the chunk takes the last key's block)
    int ku[NG], vu[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const int blk = min(base + q * CACHE_GROUP, k1 - 1) >> p.log_block;
      ku[q] = ks[blk];
      vu[q] = vs[blk];
    }
    {
      const int next = step + CD_STAGES - 1;
      int ns = slot + CD_STAGES - 1;
      if (ns >= CD_STAGES) ns -= CD_STAGES;
      if (next < steps) issue(next, ns);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(CD_STAGES - 1) : "memory");
    __syncwarp();

    // ---- scores ----
    float s[NG][4];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      int hi[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      s[q][0] = s[q][1] = s[q][2] = s[q][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        uint32_t w0[4], w1[4];
        lds128(st + ka[c] + (q * CACHE_GROUP) * HD, w0);
        lds128(st + ka[c] + (q * CACHE_GROUP + 8) * HD, w1);
        if constexpr (FMT == CACHE_E4M3) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma_f16(s[q], e4m3_half2((uint16_t)(w0[i] & 0xffffu)), e4m3_half2((uint16_t)(w1[i] & 0xffffu)),
                    e4m3_half2((uint16_t)(w0[i] >> 16)), e4m3_half2((uint16_t)(w1[i] >> 16)), qb[c][i][0],
                    qb[c][i][1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            mma_int8<false>(hi, w0[i], w1[i], w0[i + 1], w1[i + 1], qb[c][i][0], qb[c][i + 1][0]);
            mma_int8<true>(mid, w0[i], w1[i], w0[i + 1], w1[i + 1], qb[c][i][1], qb[c][i + 1][1]);
            mma_int8<true>(lo, w0[i], w1[i], w0[i + 1], w1[i + 1], qb[c][i][QW - 1], qb[c][i + 1][QW - 1]);
          }
        }
      }
      if constexpr (FMT == CACHE_INT8) {
        // |hi| <= 2^21 is exact; |256 mid + lo| < 2^31 and its rounding is 2^-24 of it
#pragma unroll
        for (int e = 0; e < 4; ++e) s[q][e] = fmaf((float)hi[e], 65536.f, (float)(mid[e] * 256 + lo[e]));
      }
    }
    // ---- weights ----
    float ve[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const float kf = cache_scale(ku[q]);
      ve[q] = vu[q] == 255 ? __uint_as_float(0x7fc00000u) : (float)(vu[q] - 127);
      const float2 f = mul2(make_float2(sl[0], sl[1]), make_float2(kf, kf));
      const float2 x = mul2(make_float2(s[q][0], s[q][1]), f), y = mul2(make_float2(s[q][2], s[q][3]), f);
      s[q][0] = x.x;
      s[q][1] = x.y;
      s[q][2] = y.x;
      s[q][3] = y.y;
    }
    if (base < k0 || base + KEYS > k1) {
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = base + q * CACHE_GROUP + 8 * e + g;
          if (key < k0 || key >= k1) s[q][2 * e] = s[q][2 * e + 1] = -INFINITY;
        }
    }
    // the maxima move seldom: only when some lane's own maximum is above them do the
    // lanes agree on new ones and is the state brought to them
    float mx[2], rx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = rx[h] = -INFINITY;
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const float x = fmaxf(s[q][h], s[q][2 + h]);
        mx[h] = fmaxf(mx[h], x);
        rx[h] = fmaxf(rx[h], x + ve[q]);
      }
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1] || rx[0] > r[0] || rx[1] > r[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], d));
          rx[h] = fmaxf(rx[h], __shfl_xor_sync(0xffffffffu, rx[h], d));
        }
        const float mn = fmaxf(m[h], mx[h]), rn = fmaxf(r[h], rx[h]);
        const float am = m[h] == mn ? 1.f : fast_exp2(m[h] - mn), ar = r[h] == rn ? 1.f : fast_exp2(r[h] - rn);
        m[h] = mn;
        r[h] = rn;
        l[h] *= am;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          o[j][h] *= ar;
          o[j][2 + h] *= ar;
        }
      }
    }
    const float2 mu = make_float2(m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]);
    const float2 ru = make_float2(r[0] == -INFINITY ? CD_SHIFT : CD_SHIFT - r[0],
                                  r[1] == -INFINITY ? CD_SHIFT : CD_SHIFT - r[1]);
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const float2 off = add2(make_float2(ve[q], ve[q]), ru);
      float pw[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 x = make_float2(s[q][2 * e], s[q][2 * e + 1]);
        const float2 a = add2(x, mu), c = add2(x, off);
        const float2 w = add2(make_float2(l[0], l[1]), make_float2(fast_exp2(a.x), fast_exp2(a.y)));
        l[0] = w.x;
        l[1] = w.y;
        pw[2 * e] = fast_exp2(c.x);
        pw[2 * e + 1] = fast_exp2(c.y);
      }
      const uint32_t b0 = movmatrix_t(pack_f16x2(pw[0], pw[1]));
      const uint32_t b1 = movmatrix_t(pack_f16x2(pw[2], pw[3]));
      // ---- values ----
      uint32_t v[4][VW];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t addr = st + va[e & 1] + (q * CACHE_GROUP + 8 * (e >> 1)) * HD;
        if constexpr (VW == 4) lds128(addr, v[e]);
        else lds64(addr, v[e]);
      }
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        uint32_t ab[4], cd[4];
        cache_zip<FMT>(v[0][i], v[1][i], ab);
        cache_zip<FMT>(v[2][i], v[3][i], cd);
        mma_f16(o[2 * i], ab[0], ab[1], cd[0], cd[1], b0, b1);
        mma_f16(o[2 * i + 1], ab[2], ab[3], cd[2], cd[3], b0, b1);
      }
    }
    __syncwarp();  // the slot may be refilled
    if (++slot == CD_STAGES) slot = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- merge the warps through shared memory (their rings are done with) ----
  __syncthreads();
  float* red_o = reinterpret_cast<float*>(cd_ring);  // [CD_WARPS][8][HD]
  float* red_s = red_o + CD_WARPS * 8 * HD;          // [CD_WARPS][3][8]
  static_assert(cd_smem<HD>() >= (CD_WARPS * 8 * HD + CD_WARPS * 24) * 4, "merge buffers fit in the rings");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
    if (g == 0) {
      red_s[warp * 24 + 2 * t + h] = m[h];
      red_s[warp * 24 + 8 + 2 * t + h] = l[h];
      red_s[warp * 24 + 16 + 2 * t + h] = r[h];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      red_o[(warp * 8 + 2 * t + h) * HD + HD / 8 * g + 2 * j] = o[j][h];
      red_o[(warp * 8 + 2 * t + h) * HD + HD / 8 * g + 2 * j + 1] = o[j][2 + h];
    }
  }
  __syncthreads();
  // this chunk's partial: to global memory, or (CLU) to own[8][4 + HD]
  float* own = red_s + CD_WARPS * 24;
  const long long hstride = CLU ? 4 + HD : (long long)S.n_launched * (4 + HD);
  float* part0 =
      CLU ? own : S.partials + ((long long)(b * p.H + hk * G) * S.n_launched + chunk) * (4 + HD);
  for (int idx = threadIdx.x; idx < G * HD; idx += CD_THREADS) {
    const int h = idx / HD, d = idx - h * HD;
    float M = -INFINITY, R = -INFINITY;
#pragma unroll
    for (int w = 0; w < CD_WARPS; ++w) {
      M = fmaxf(M, red_s[w * 24 + h]);
      R = fmaxf(R, red_s[w * 24 + 16 + h]);
    }
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < CD_WARPS; ++w) {
      if (red_s[w * 24 + 8 + h] == 0.f) continue;  // no key of this warp counts
      L += red_s[w * 24 + 8 + h] * fast_exp2(red_s[w * 24 + h] - M);
      O += red_o[(w * 8 + h) * HD + d] * fast_exp2(red_s[w * 24 + 16 + h] - R);
    }
    float* part = part0 + h * hstride;
    part[4 + d] = O;
    if (d == 0) {
      part[0] = M;
      part[1] = L;
      part[2] = R;
    }
  }
  if constexpr (CLU) {
    static_assert(cd_smem<HD>() >= (CD_WARPS * 8 * HD + CD_WARPS * 24 + 8 * (4 + HD)) * 4, "partial fits behind them");
    __syncwarp();
    cluster_sync();
    // items of 32 columns of one row of one set, dealt to the cluster's warps
    constexpr int COLS = HD / 32;
    const int nct = (int)cluster_nctarank();
    const int sets = (p.out[0] ? 1 : 0) + (p.out[1] ? 1 : 0);
    const uint32_t mine = smem_u32(own);
    for (int item = (int)cluster_ctarank() * CD_WARPS + warp; item < sets * G * COLS; item += nct * CD_WARPS) {
      const int set = p.out[0] ? item / (G * COLS) : 1, row = item / COLS % G, d = item % COLS * 32 + lane;
      const int r0 = set ? n_dense : 0, n = p.set[set].n_launched;
      const uint32_t at = mine + row * (4 + HD) * 4;
      float ov[CD_CLUSTER_MAX];
#pragma unroll
      for (int x = 0; x < CD_CLUSTER_MAX; ++x)
        ov[x] = x < n ? ld_dsmem_f32(dsmem_addr(at + (4 + d) * 4, r0 + x)) : 0.f;
      float hm = -INFINITY, hl = 0.f, hr = -INFINITY;
      if (lane < n) {
        const uint32_t head = dsmem_addr(at, r0 + lane);
        hm = ld_dsmem_f32(head);
        hl = ld_dsmem_f32(head + 4);
        hr = ld_dsmem_f32(head + 8);
      }
      MergeState<1> st;
      st.start();
      const float hms[1] = {hm}, hls[1] = {hl}, hrs[1] = {hr};
      float wo[1];
      st.weigh(hms, hls, hrs, wo);
      float acc[MG_ROWS] = {};
#pragma unroll
      for (int x = 0; x < CD_CLUSTER_MAX; ++x) merge_add(acc[x % MG_ROWS], ov[x], __shfl_sync(0xffffffffu, wo[0], x));
#pragma unroll
      for (int y = 1; y < MG_ROWS; ++y) acc[0] += acc[y];
      p.out[set][(long long)(b * p.H + hk * G + row) * HD + d] = st.finish(acc[0]);
    }
    __syncwarp();
    cluster_sync();  // no CTA exits while a peer may still read its partial
  }
}

// Merge of a key set's partials: grid (B * H, key sets), MG_ROWS threads per head
// dim.  The threads' columns of the first MG_ROWS * MG_LOADS chunks and their headers
// are fetched at once, so a set of up to that many chunks costs one round trip to L2.
// A programmatic dependent launch: its CTAs are resident when the partials' grid ends.
template <int HD>
__global__ void __launch_bounds__(MG_ROWS* HD) cache_merge_kernel(const __grid_constant__ CacheDecodeParams p) {
  constexpr int TILE = MG_ROWS * MG_LOADS, HEADS = TILE / 32;
  static_assert(HD % 32 == 0 && TILE % 32 == 0, "a warp's lanes hold one tile's headers and share a row");
  __shared__ float red[MG_ROWS][HD];
  const int bh = blockIdx.x, which = p.out[0] ? blockIdx.y : 1;
  const int d = threadIdx.x % HD, y = threadIdx.x / HD, lane = threadIdx.x & 31;
  const CacheDecodeSet& S = p.set[which];
  const float* base = S.partials + (long long)bh * S.n_launched * (4 + HD);
  grid_dependency_wait();
  MergeState<HEADS> st;
  st.start();
  float O = 0.f;
  for (int x0 = 0; x0 < S.n_launched; x0 += TILE) {
    const int n = min(TILE, S.n_launched - x0);
    const float* tile = base + (long long)x0 * (4 + HD);
    float ov[MG_LOADS];
#pragma unroll
    for (int i = 0; i < MG_LOADS; ++i) {
      const int x = y + i * MG_ROWS;
      ov[i] = x < n ? tile[(long long)x * (4 + HD) + 4 + d] : 0.f;
    }
    float hm[HEADS], hl[HEADS], hr[HEADS], wo[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
      const int x = lane + 32 * k;
      float4 h = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      if (x < n) h = *reinterpret_cast<const float4*>(tile + (long long)x * (4 + HD));
      hm[k] = h.x;
      hl[k] = h.y;
      hr[k] = h.z;
    }
    O *= st.weigh(hm, hl, hr, wo);
#pragma unroll
    for (int i = 0; i < MG_LOADS; ++i)
      merge_add(O, ov[i], __shfl_sync(0xffffffffu, wo[i * MG_ROWS / 32], (y + i * MG_ROWS) & 31));
  }
  red[y][d] = O;
  __syncthreads();
  if (y == 0) {
#pragma unroll
    for (int i = 1; i < MG_ROWS; ++i) O += red[i][d];
    p.out[which][(long long)bh * HD + d] = st.finish(O);
  }
}

// Sets the kernel's launch attributes on the current device, once per device (they
// stay set); for a cluster size, *active is how many such clusters are resident at once.
template <int HD, int FMT, bool CLU>
static cudaError_t prepare_kernel(int nct, int* active) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static std::atomic<int> state[kDevices][CD_CLUSTER_MAX + 1];  // 0 unknown, else 1 + clusters
  auto kernel = cache_decode_kernel<HD, FMT, CLU>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kDevices) return cudaErrorInvalidDevice;
  std::atomic<int>& st = state[dev][CLU ? nct : 0];
  if (st.load(std::memory_order_acquire) == 0) {
    std::lock_guard<std::mutex> lock(mu);
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, cd_smem<HD>());
    if (e == cudaSuccess && CLU) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    int n = 1;
    if (CLU) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, nct);
      cfg.blockDim = dim3(CD_THREADS);
      cfg.dynamicSmemBytes = cd_smem<HD>();
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.y = nct;
      attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();  // a refused size is not an error of the call
        n = 0;
      }
    }
    st.store(1 + n, std::memory_order_release);
  }
  *active = st.load(std::memory_order_acquire) - 1;
  return cudaSuccess;
}

template <int HD, int FMT, bool CLU>
static cudaError_t launch_partials(const CacheDecodeParams& p, int nct, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.B * p.Hkv, nct);
  cfg.blockDim = dim3(CD_THREADS);
  cfg.dynamicSmemBytes = cd_smem<HD>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.y = nct;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLU ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, cache_decode_kernel<HD, FMT, CLU>, p);
}

template <int HD, int FMT>
static cudaError_t decode_as(const CacheDecodeParams& p, cudaStream_t stream) {
  int nct = 0;
  for (int which = 0; which < 2; ++which)
    if (p.out[which]) nct += p.set[which].n_launched;
  int active = 0;
  cudaError_t e;
  if (p.clusters && nct <= CD_CLUSTER_MAX) {
    // Clusters save the merge launch (2.5 us of host time, 0.3 us of the GPU's) where
    // they are all resident at once.  A cluster's CTAs lie in one GPC, so fewer are than
    // of single CTAs, and a second wave costs more than the launch: 123 us for 83 with
    // 32 clusters of 9 at 4 x 65536 keys.
    if ((e = prepare_kernel<HD, FMT, true>(nct, &active)) != cudaSuccess) return e;
    if ((long long)p.B * p.Hkv <= active) return launch_partials<HD, FMT, true>(p, nct, stream);
  }
  if ((e = prepare_kernel<HD, FMT, false>(0, &active)) != cudaSuccess) return e;
  if ((e = launch_partials<HD, FMT, false>(p, nct, stream)) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.B * p.H, (p.out[0] ? 1 : 0) + (p.out[1] ? 1 : 0));
  cfg.blockDim = dim3(MG_ROWS * HD);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cache_merge_kernel<HD>, p);
}

cudaError_t launch_cache_decode(const CacheDecodeParams& p, int head_dim, int format, cudaStream_t stream) {
  if (head_dim == 128)
    return format == CACHE_E4M3 ? decode_as<128, CACHE_E4M3>(p, stream) : decode_as<128, CACHE_INT8>(p, stream);
  return format == CACHE_E4M3 ? decode_as<64, CACHE_E4M3>(p, stream) : decode_as<64, CACHE_INT8>(p, stream);
}

}  // namespace dta
