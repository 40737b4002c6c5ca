// extern "C" entry points of the 8-bit KV cache: argument validation, the
// split of a decode call into chunks, and the launches.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "delta_attention_b200.h"
#include "dta_cache.h"
#include "dta_internal.h"

namespace {

inline bool aligned(const void* p, unsigned a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline bool stride16(long long s, int bytes) { return s > 0 && (s * bytes) % 16 == 0; }
inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Shapes, strides and pointers of a cache; *log_block and the two sides.
int check_cache(const dta_cache_desc& c, int* log_block, dta::CacheSide side[2]) {
  if (c.batch <= 0 || c.n_kv_heads <= 0 || c.capacity <= 0 || c.capacity > (1 << 30)) return DTA_ERR_SHAPE;
  if (c.head_dim != 64 && c.head_dim != 128) return DTA_ERR_HEAD_DIM;
  // the kernels' grid y is batch x KV head (at most 65535)
  if ((long long)c.batch * c.n_kv_heads > 65535) return DTA_ERR_SHAPE;
  if (c.block != 16 && c.block != 32 && c.block != 64 && c.block != 128) return DTA_ERR_INVALID_ARG;
  if (c.format != DTA_CACHE_E4M3 && c.format != DTA_CACHE_INT8) return DTA_ERR_INVALID_ARG;
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return DTA_ERR_INVALID_ARG;
  if (!aligned(c.k, 16) || !aligned(c.v, 16)) return DTA_ERR_ALIGNMENT;
  for (long long s : {(long long)c.k_stride_b, (long long)c.k_stride_h, (long long)c.k_stride_s,
                      (long long)c.v_stride_b, (long long)c.v_stride_h, (long long)c.v_stride_s})
    if (!stride16(s, 1)) return DTA_ERR_STRIDE;
  for (long long s : {(long long)c.k_scale_stride_b, (long long)c.k_scale_stride_h, (long long)c.v_scale_stride_b,
                      (long long)c.v_scale_stride_h})
    if (s <= 0) return DTA_ERR_STRIDE;
  *log_block = c.block == 16 ? 4 : c.block == 32 ? 5 : c.block == 64 ? 6 : 7;
  side[0] = {reinterpret_cast<uint8_t*>(c.k), c.k_stride_b, c.k_stride_h, c.k_stride_s, c.k_scale,
             c.k_scale_stride_b, c.k_scale_stride_h};
  side[1] = {reinterpret_cast<uint8_t*>(c.v), c.v_stride_b, c.v_stride_h, c.v_stride_s, c.v_scale,
             c.v_scale_stride_b, c.v_scale_stride_h};
  return DTA_OK;
}

bool type_ok(int t) { return t == DTA_CACHE_BF16 || t == DTA_CACHE_FP16 || t == DTA_CACHE_FP32; }

// An optional device list of one element or one per sequence; *step its stride.
int check_list(const int32_t* list, int n, int batch, int* step) {
  *step = 0;
  if (!list) return DTA_OK;
  if (!aligned(list, 4)) return DTA_ERR_ALIGNMENT;
  if (n != 1 && n != batch) return DTA_ERR_SHAPE;
  *step = n == 1 ? 0 : 1;
  return DTA_OK;
}

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

constexpr int kRampSteps = dta::CACHE_RAMP_STEPS;
constexpr int kMaxSms = 160;  // SMs that are counted at most (a B200 has 148)

// CTAs of the partial kernel that are resident on an SM (shared memory bounds them).
constexpr int kResidentCtas = 2;

// Chunk of the sparse set, by the estimated time of its CTAs in steps: one that all are
// resident with costs its own steps and kRampSteps; more of them the sum of their
// costs over the slots and half a chunk's for the end; beyond 16 chunks per unit a
// merge launch, two steps.  (128 + 2048 keys, 8 units: 6.0 us with 256-key chunks, 6.4 with
// 384.)  It goes by the sink and window (each at most the call's n_keys), the units, the head
// size and the device's SMs, not by the dense set or a device key count: on one device, calls
// with the same n_keys cut a sparse row alike, with and without the dense one.  Calls
// whose n_keys differ and lie below the sink or window may cut it differently (a host count,
// and the capacity with that count on the device): those rows differ by rounding.
constexpr int kSparseSteps[] = {1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32};
constexpr int kSparseWaves = 4;  // chunks that would take more waves are not tried
constexpr long long kSparseKeys = 1 << 23;  // windows beyond this take longer chunks (a launch has 65535 at most)

int sparse_chunk(long long sink, long long window, long long units, long long slots, int step) {
  const long long f = sink + window > kSparseKeys ? ceil_div(sink + window, kSparseKeys) : 1;
  const long long longest = f * kSparseSteps[sizeof(kSparseSteps) / sizeof(int) - 1];
  long long best = longest, best_cost = -1;
  for (int st : kSparseSteps) {
    const long long steps = f * st, c = steps * step, k = ceil_div(sink, c) + ceil_div(window, c);
    if (units * k > kSparseWaves * slots && steps != longest) continue;
    const long long sum = ceil_div(sink, step) + ceil_div(window, step) + k * kRampSteps;
    const long long own = steps + kRampSteps;  // (costs count half steps)
    const long long cost = (units * k <= slots ? 2 * own : 2 * units * sum / slots + own) + (k > 16 ? 4 : 0);
    if (best_cost < 0 || cost < best_cost) {
      best = steps;
      best_cost = cost;
    }
  }
  return (int)best * step;
}
// At most this many sparse chunks of all units, on any device and for any smaller sink and window.
long long sparse_chunks_max(long long sink, long long window, long long units) {
  const long long few = (long long)kSparseWaves * kMaxSms * kResidentCtas;
  const long long chunks = ceil_div(sink + window, 32 * 128), most = kSparseKeys / (32 * 128);
  const long long many = units * ((chunks < most ? chunks : most) + 2);
  return few > many ? few : many;
}

// Chunk of the dense set: the one with the least estimated time, in steps of a CTA.
// 7/8 of the resident CTAs are used (the sparse ones take the rest where they are
// wanted): the memory is saturated by them, and SMs that have one CTA instead of two
// even out at the end (131072 keys, 8 KV heads: 47.1 us with 256 CTAs, 48.6 with 296, 55
// with 168; 4 x 65536: 82.1 with 256, 88.8 with 288, 92 with 192).  With that many
// `slots`, w waves of them take k = w slots / units chunks of each unit (a (batch, KV
// head)); a CTA costs its chunk's steps plus kRampSteps for its start and end (a step
// takes 1.5 us while the memory is saturated).  The sparse set's CTAs, if they are wanted
// too, come last: into the places that the dense ones leave, else after them, so fewer
// chunks that leave them room are tried as well.  Where sequences have lengths of their
// own, about half of the chunks are taken to be empty.  (16 sequences of 8191 down to 0
// keys, 8 KV heads: 29.6 us with 2048-key chunks, 32.6 with 1024, 38.3 with 4096.  32761
// keys, 8 KV heads of 8 queries, both rows: 21.5 us with 1152, which leaves the sparse
// chunks room, 25.1 with 896.)
constexpr int kWaves = 4;

int dense_chunk(long long n, long long units, long long sparse_ctas, long long sparse_steps, bool ragged,
                long long slots, int step) {
  if (n <= step) return step;
  if (sparse_ctas == 0 && slots > 1) slots = slots * 7 / 8;
  const long long sparse_cost = sparse_steps + kRampSteps;
  long long best = 0, best_cost = 0;
  for (int i = 0; i < 3 * kWaves; ++i) {
    if (sparse_ctas == 0 && i % 3 != 0) continue;
    const long long room = i % 3 * (sparse_ctas < slots / 2 ? sparse_ctas : slots / 2) / 2;
    const long long places = (i / 3 + 1) * slots - room, k = places / units > 0 ? places / units : 1;
    const long long steps = ceil_div(n, k * step), cost = steps + kRampSteps;
    const long long ctas = ceil_div(ceil_div(n, steps * step) * units, ragged ? 2 : 1);
    const long long waves = ceil_div(ctas, slots);
    const long long beside = (waves * slots - ctas) * (cost / sparse_cost);
    const long long after = sparse_ctas > beside ? ceil_div(sparse_ctas - beside, slots) * sparse_cost : 0;
    const long long total = waves * cost + after;
    if (best == 0 || total < best_cost) {
      best = steps * step;
      best_cost = total;
    }
  }
  return (int)best;
}

// At most this many dense chunks per unit, on any device.
long long dense_chunks_max(long long n, long long units, int step) {
  const long long k = (long long)kWaves * kMaxSms * kResidentCtas / units;
  const long long shortest = n > 0 ? ceil_div(n, step) : 1;  // (without keys: one empty chunk)
  return k < 1 ? 1 : k < shortest ? k : shortest;
}

// Checks the arguments (no CUDA call) and fills in all but the plan.
int decode_setup(const dta_cache_decode_args* a, dta::CacheDecodeParams* p) {
  if (!a || a->abi_version != DTA_ABI_VERSION) return DTA_ERR_INVALID_ARG;
  memset(p, 0, sizeof(*p));
  const dta_cache_desc& c = a->cache;
  int st = check_cache(c, &p->log_block, p->side);
  if (st != DTA_OK) return st;
  if (a->n_heads <= 0 || a->n_heads % c.n_kv_heads != 0 || a->n_heads / c.n_kv_heads > 8) return DTA_ERR_SHAPE;
  if (a->n_keys < 0 || a->n_keys > c.capacity) return DTA_ERR_SHAPE;
  if (a->window < 0 || a->sink < 0) return DTA_ERR_INVALID_ARG;
  if ((st = check_list(a->n_keys_dev, a->n_lengths, c.batch, &p->len_step)) != DTA_OK) return st;
  p->B = c.batch; p->H = a->n_heads; p->Hkv = c.n_kv_heads; p->G = a->n_heads / c.n_kv_heads;
  p->n_keys = a->n_keys;
  p->n_keys_dev = a->n_keys_dev;
  p->scale_log2 = a->scaling * 1.4426950408889634f;
  // sink and window beyond the cache mean the whole cache
  p->window = a->window < a->n_keys ? a->window : a->n_keys;
  p->sink = a->sink < a->n_keys ? a->sink : a->n_keys;
  return DTA_OK;
}

// The chunks of the sets that are wanted, for a device of `sms` SMs.
void decode_plan(const dta_cache_decode_args* a, dta::CacheDecodeParams* p, int sms) {
  const long long units = (long long)p->B * p->Hkv, n = p->n_keys;
  const long long slots = (sms < kMaxSms ? sms : kMaxSms) * kResidentCtas;
  const int step = dta::cache_step(a->cache.head_dim);
  const bool ragged = p->n_keys_dev && p->len_step;
  p->clusters = !(ragged && a->dense_out);  // an empty chunk would hold its place until its cluster is done
  if (a->sparse_out) {
    const int c = sparse_chunk(p->sink, p->window, units, slots, step);
    p->set[1].chunk = c;
    p->set[1].n_sink_chunks = (int)ceil_div(p->sink, c);
    p->set[1].n_launched = p->set[1].n_sink_chunks + (int)ceil_div(p->window, c);
    if (p->set[1].n_launched < 1) p->set[1].n_launched = 1;  // no keys: one empty partial
  }
  if (a->dense_out) {
    const int c = dense_chunk(n, units, units * p->set[1].n_launched, p->set[1].chunk / step, ragged, slots, step);
    p->set[0].chunk = c;
    p->set[0].n_launched = n > 0 ? (int)ceil_div(n, c) : 1;
  }
}

// Bytes of the partials of `chunks` chunks (of all units together), each of a unit's query heads.
size_t partial_bytes(const dta_cache_decode_args* a, long long chunks) {
  return align_up((size_t)chunks * (a->n_heads / a->cache.n_kv_heads) * (4 + a->cache.head_dim) * 4, 256);
}

}  // namespace

extern "C" {

int dta_cache_write(const dta_cache_write_args* a, void* stream) {
  if (!a || a->abi_version != DTA_ABI_VERSION) return DTA_ERR_INVALID_ARG;
  dta::CacheWriteParams p;
  memset(&p, 0, sizeof(p));
  const dta_cache_desc& c = a->cache;
  int st = check_cache(c, &p.log_block, p.side);
  if (st != DTA_OK) return st;
  if (!type_ok(a->src_type)) return DTA_ERR_INVALID_ARG;
  if (a->n_new < 0 || a->n_new > c.capacity) return DTA_ERR_SHAPE;
  if (!a->pos_dev && (a->pos < 0 || a->pos > c.capacity - a->n_new)) return DTA_ERR_SHAPE;
  if ((st = check_list(a->pos_dev, a->n_pos, c.batch, &p.pos_step)) != DTA_OK) return st;
  if ((st = check_list(a->lengths, a->n_lengths, c.batch, &p.len_step)) != DTA_OK) return st;
  if (a->error_word && !aligned(a->error_word, 4)) return DTA_ERR_ALIGNMENT;
  if (a->n_new == 0) return DTA_OK;
  if (!a->k_new || !a->v_new) return DTA_ERR_INVALID_ARG;
  if (!aligned(a->k_new, 16) || !aligned(a->v_new, 16)) return DTA_ERR_ALIGNMENT;
  const int es = a->src_type == DTA_CACHE_FP32 ? 4 : 2;
  const int64_t str[2][3] = {{a->k_new_stride_b, a->k_new_stride_h, a->k_new_stride_s},
                             {a->v_new_stride_b, a->v_new_stride_h, a->v_new_stride_s}};
  for (int i = 0; i < 2; ++i) {
    for (int64_t s : str[i])
      if (!stride16(s, es)) return DTA_ERR_STRIDE;
    p.src[i] = i ? a->v_new : a->k_new;
    p.src_sb[i] = str[i][0]; p.src_sh[i] = str[i][1]; p.src_ss[i] = str[i][2];
  }
  int sms = 0;
  if ((st = dta::check_device(&sms)) != DTA_OK) return st;
  p.Hkv = c.n_kv_heads; p.n_new = a->n_new; p.capacity = c.capacity;
  p.pos = a->pos; p.pos_dev = a->pos_dev; p.lengths = a->lengths; p.error_word = a->error_word;
  const cudaError_t e = dta::launch_cache_write(p, c.batch, c.head_dim, c.format, a->src_type,
                                                reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? (int)DTA_OK : dta::fail_cuda(e);
}

int dta_cache_read(const dta_cache_read_args* a, void* stream) {
  if (!a || a->abi_version != DTA_ABI_VERSION) return DTA_ERR_INVALID_ARG;
  dta::CacheReadParams p;
  memset(&p, 0, sizeof(p));
  const dta_cache_desc& c = a->cache;
  int st = check_cache(c, &p.log_block, p.side);
  if (st != DTA_OK) return st;
  if (!type_ok(a->dst_type)) return DTA_ERR_INVALID_ARG;
  if (a->start < 0 || a->n_keys < 0 || a->start > c.capacity || a->n_keys > c.capacity - a->start) return DTA_ERR_SHAPE;
  if ((st = check_list(a->lengths, a->n_lengths, c.batch, &p.len_step)) != DTA_OK) return st;
  if (a->n_keys == 0) return DTA_OK;
  if (!a->out_k || !a->out_v) return DTA_ERR_INVALID_ARG;
  if (!aligned(a->out_k, 16) || !aligned(a->out_v, 16)) return DTA_ERR_ALIGNMENT;
  int sms = 0;
  if ((st = dta::check_device(&sms)) != DTA_OK) return st;
  p.dst[0] = a->out_k; p.dst[1] = a->out_v;
  p.Hkv = c.n_kv_heads; p.n = a->n_keys; p.start = a->start; p.lengths = a->lengths;
  const cudaError_t e = dta::launch_cache_read(p, c.batch, c.head_dim, c.format, a->dst_type,
                                               reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? (int)DTA_OK : dta::fail_cuda(e);
}

// Both key sets' partials, whichever outputs the call asks for: enough for any
// device, and never less for more keys (a caller may size it for the capacity once).
size_t dta_cache_decode_workspace_size(const dta_cache_decode_args* a) {
  dta::CacheDecodeParams p;
  if (decode_setup(a, &p) != DTA_OK) return 0;
  const long long units = (long long)p.B * p.Hkv;
  return partial_bytes(a, units * dense_chunks_max(a->n_keys, units, dta::cache_step(a->cache.head_dim))) +
         partial_bytes(a, sparse_chunks_max(p.sink, p.window, units));
}

int dta_cache_decode(const dta_cache_decode_args* a, void* stream) {
  dta::CacheDecodeParams p;
  int st = decode_setup(a, &p);
  if (st != DTA_OK) return st;
  if (!a->q || (!a->dense_out && !a->sparse_out)) return DTA_ERR_INVALID_ARG;
  if (!aligned(a->q, 16) || !aligned(a->dense_out, 16) || !aligned(a->sparse_out, 16)) return DTA_ERR_ALIGNMENT;
  if (!stride16(a->q_stride_b, 2) || !stride16(a->q_stride_h, 2)) return DTA_ERR_STRIDE;
  const size_t need = dta_cache_decode_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)) return DTA_ERR_WORKSPACE;
  int sms = 0;
  if ((st = dta::check_device(&sms)) != DTA_OK) return st;
  decode_plan(a, &p, sms);
  p.q = reinterpret_cast<const __nv_bfloat16*>(a->q);
  p.q_sb = a->q_stride_b; p.q_sh = a->q_stride_h;
  p.set[0].partials = reinterpret_cast<float*>(a->workspace);
  p.set[1].partials = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) +
                                                 partial_bytes(a, (long long)p.B * p.Hkv * p.set[0].n_launched));
  p.out[0] = reinterpret_cast<__nv_bfloat16*>(a->dense_out);
  p.out[1] = reinterpret_cast<__nv_bfloat16*>(a->sparse_out);
  const cudaError_t e = dta::launch_cache_decode(p, a->cache.head_dim, a->cache.format,
                                                 reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? (int)DTA_OK : dta::fail_cuda(e);
}

}  // extern "C"
