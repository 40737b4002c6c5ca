// Internal launch parameters of the 8-bit KV-cache kernels (not part of the C ABI).
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <stdint.h>

namespace dta {

// Element types of dta_cache_write_args.src_type / dta_cache_read_args.dst_type.
enum : int { CACHE_BF16 = 0, CACHE_FP16 = 1, CACHE_FP32 = 2 };
// Code formats of the cache.
enum : int { CACHE_E4M3 = 0, CACHE_INT8 = 1 };

// One of the two code tensors (K or V): codes [b, Hkv, capacity, d] with strides
// in bytes, biased exponents of the block scales [b, Hkv, blocks].
struct CacheSide {
  uint8_t* codes;
  long long sb, sh, ss;
  uint8_t* scale;
  long long scale_sb, scale_sh;
};

struct CacheWriteParams {
  const void* src[2];                 // K, V rows
  long long src_sb[2], src_sh[2], src_ss[2];  // in elements
  CacheSide side[2];
  int Hkv, n_new, capacity, log_block;
  int pos;
  const int* pos_dev;                 // optional; element b * pos_step
  int pos_step;
  const int* lengths;                 // optional; element b * len_step
  int len_step;
  int* error_word;
};

struct CacheReadParams {
  CacheSide side[2];
  void* dst[2];                       // [b, Hkv, n, d] contiguous
  int Hkv, n, start, log_block;
  const int* lengths;                 // optional live key counts; element b * len_step
  int len_step;
};

// The key sets of a decode call are cut into chunks, one per CTA.  Chunk bounds
// lie on multiples of CACHE_GROUP keys (absolute), which never straddle a scale
// block; only a key set's own first and last key may lie inside a group.
constexpr int CACHE_GROUP = 16;

// Keys in one step of a CTA of the decode kernel, and what its start and end cost, in steps.
constexpr int cache_step(int head_dim) { return head_dim == 128 ? 128 : 256; }
constexpr int CACHE_RAMP_STEPS = 3;

struct CacheDecodeSet {
  int chunk;               // keys per chunk, a multiple of CACHE_GROUP
  int n_sink_chunks;       // sparse set: chunks that cover [0, sink)
  int n_launched;
  float* partials;         // [b, H, n_launched, 4 + d]: (m, l, r, -, o[d]) per chunk
};

struct CacheDecodeParams {
  const __nv_bfloat16* q;
  long long q_sb, q_sh;
  CacheSide side[2];
  int B, H, Hkv, G, n_keys, log_block;
  const int* n_keys_dev;   // optional live key counts; element b * len_step
  int len_step;
  float scale_log2;
  int window, sink;
  int clusters;            // whether chunks may merge within a cluster
  CacheDecodeSet set[2];   // 0: dense, 1: sparse
  __nv_bfloat16* out[2];   // dense, sparse; either may be null
};

cudaError_t launch_cache_write(const CacheWriteParams& p, int batch, int head_dim, int format, int src_type,
                               cudaStream_t stream);
cudaError_t launch_cache_read(const CacheReadParams& p, int batch, int head_dim, int format, int dst_type,
                              cudaStream_t stream);
cudaError_t launch_cache_decode(const CacheDecodeParams& p, int head_dim, int format, cudaStream_t stream);

}  // namespace dta
