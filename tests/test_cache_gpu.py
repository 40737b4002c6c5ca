"""GPU parity of the 8-bit KV cache (cache_write, cache_read, cache_decode) with
the 64-bit oracle.

Writing and reading are exact: scales are powers of two, so a code is one
rounding of an exact product and must equal the oracle's, bit for bit.

Attention is held to, per output element with weights w, W = sum w |v| and
off_j = scaling * (c |q| . |k_j| + e max|q| sum|k_j|):
  2^-8 |out|             the output's rounding to bf16 (half a step)
  2^-11 W                the weights' rounding to fp16
  n 2^-38 max|v|         weights below fp16's normal range (half a step is 2^-25 of 2^14, over l >= 1)
  sum w off |v| + (sum w off) W   the scores, off by off_j, move a weight and the sum of the weights
                         relatively by as much.  c = (d + 6) 2^-23: sums over d terms in fp32 (d steps,
                         and 6 more for the products with the scales and log2 e).  e: the query's own
                         rounding, 2^-29 for e4m3 (fp16, scaled) and 1/65024 for int8 (half a step of 1/32512)
  2^-13 W                sums of weights and products in fp32 (at most 2^9 steps of 2^-23 each in a warp's
                         share, and the merges), exp2's 2^-22, the maxima's shifts
"""

import math

import pytest
import torch

from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def _ops():
    from delta_attention_b200 import ops
    return ops


def _cache(b, h, cap, d, fmt, block, pad=0, seed=0):
    """A cache full of the codes 0..255 (NaN codes and scales among them): what
    is not written must not matter."""
    from delta_attention_b200.kv_cache import CODE_TYPES, SCALE_TYPE, QuantizedKV
    g = torch.Generator().manual_seed(seed)

    def noise(*shape):
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).cuda()

    blocks = -(-cap // block)
    k = noise(b, h, cap + pad, d + 16 * (pad > 0)).view(CODE_TYPES[fmt])[:, :, :cap, :d]
    v = noise(b, cap, h, d).view(CODE_TYPES[fmt]).transpose(1, 2) if pad else noise(b, h, cap, d).view(CODE_TYPES[fmt])
    ks, vs = noise(b, h, blocks + pad).view(SCALE_TYPE)[:, :, :blocks], noise(b, h, blocks).view(SCALE_TYPE)
    return QuantizedKV(k, v, ks, vs, block)


def _state(cache):
    """[(codes float64, scale bytes int64)] of K and V on the CPU."""
    return [(c.float().cpu().double(), s.view(torch.uint8).cpu().long())
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


def _raw(cache):
    return [t.view(torch.uint8).cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def _rows(b, h, t, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, h, t, d, generator=g) * torch.exp(spread * torch.randn(b, h, t, 1, generator=g))
    return x.to(dtype)


def _expect(state, new, pos, lengths, block, fmt):
    for (codes, scale), x in zip(state, new):
        for i in range(x.shape[0]):
            for h in range(x.shape[1]):
                orc.write_rows(codes[i, h], scale[i, h], x[i, h, :lengths[i]], pos[i], block, fmt)


def _same(cache, state, upto, block):
    """Every live row's code and every live block's scale."""
    for (codes, scale), (want, wu) in zip(_state(cache), state):
        for i, n in enumerate(upto):
            assert torch.equal(scale[i, :, :-(-n // block)], wu[i, :, :-(-n // block)])
            a, w = codes[i, :, :n], want[i, :, :n]
            assert torch.equal(a.isnan(), w.isnan())
            assert torch.equal(a.nan_to_num(), w.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt,d,block", [("e4m3", 128, 64), ("int8", 64, 16), ("e4m3", 64, 128), ("int8", 128, 32),
                                         ("e4m3", 128, 16), ("int8", 128, 128)])
def test_write_and_append(fmt, d, block, dtype):
    """A prompt from position 0, then appends of odd lengths (single tokens
    among them) whose magnitudes grow, so that scales of begun blocks rise."""
    b, h, cap = 2, 3, 301
    cache = _cache(b, h, cap, d, fmt, block, seed=d + block)
    state = _state(cache)
    pos = 0
    for i, t in enumerate((133, 1, 1, 62, 1, 17, 86)):
        new = [(_rows(b, h, t, d, torch.float32, 10 * i + j) * 3.0 ** (i % 4)).to(dtype) for j in range(2)]
        _ops().cache_write(cache, new[0].cuda(), new[1].cuda(), pos=pos)
        _expect(state, new, [pos] * b, [t] * b, block, fmt)
        pos += t
        _same(cache, state, [pos] * b, block)
    assert pos == cap


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_ragged_positions_and_lengths(fmt):
    """Positions and lengths of each sequence on the device; rows that are not
    written, and blocks that are not touched, keep their bytes."""
    b, h, cap, d, block, t = 5, 2, 500, 128, 32, 70
    cache = _cache(b, h, cap, d, fmt, block, pad=2, seed=1)
    first = [_rows(b, h, 430, d, torch.bfloat16, 2 + j) for j in range(2)]
    _ops().cache_write(cache, first[0].cuda(), first[1].cuda(), pos=0)
    state, before = _state(cache), _raw(cache)
    pos, lengths = [0, 31, 64, 429, 430], [70, 1, 0, 70, 33]
    new = [_rows(b, h, t, d, torch.bfloat16, 7 + j) * 4 for j in range(2)]
    _ops().cache_write(cache, new[0].cuda(), new[1].cuda(), pos=torch.tensor(pos, dtype=torch.int32).cuda(),
                       lengths=torch.tensor(lengths, dtype=torch.int32).cuda(), check=True)
    _expect(state, new, pos, lengths, block, fmt)
    _same(cache, state, [p + n for p, n in zip(pos, lengths)], block)
    after = _raw(cache)
    for i in range(b):
        end = pos[i] + lengths[i]
        lo, hi = pos[i] // block, -(-end // block) if lengths[i] else pos[i] // block
        for x in (0, 1):
            assert torch.equal(after[x][i, :, :lo * block], before[x][i, :, :lo * block])
            assert torch.equal(after[x][i, :, end:], before[x][i, :, end:])  # behind the written rows: same bytes
        for x in (2, 3):
            assert torch.equal(after[x][i, :, :lo], before[x][i, :, :lo])
            assert torch.equal(after[x][i, :, hi:], before[x][i, :, hi:])


@pytest.mark.parametrize("pos,length", [(-1, 3), (290, 11), (301, 0), (5, 12), (5, -1), (2 ** 31 - 1, 1)])
def test_write_device_position_outside_the_cache(pos, length):
    """A device position or length outside the cache writes nothing of its
    sequence, is recorded, and leaves the other sequence's write alone."""
    from delta_attention_b200._lib import DtaError
    ops = _ops()
    cache = _cache(2, 2, 300, 64, "e4m3", 64, seed=4)
    before, state = _raw(cache), _state(cache)
    new = [_rows(2, 2, 11, 64, torch.bfloat16, 3 + j) for j in range(2)]
    ops.check_errors()
    with pytest.raises(DtaError, match="105"):
        ops.cache_write(cache, new[0].cuda(), new[1].cuda(), pos=torch.tensor([pos, 0], dtype=torch.int32).cuda(),
                        lengths=torch.tensor([length, 11], dtype=torch.int32).cuda(), check=True)
    ops.check_errors()
    for x, y in zip(_raw(cache), before):
        assert torch.equal(x[0], y[0])
    _expect([(c[1:], s[1:]) for c, s in state], [x[1:] for x in new], [0], [11], 64, "e4m3")
    for (codes, scale), (want, wu) in zip(_state(cache), state):
        assert torch.equal(codes[1, :, :11], want[1, :, :11]) and torch.equal(scale[1, :, 0], wu[1, :, 0])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_special_values(fmt):
    """Zeros, subnormals, the largest magnitudes, values on the border of a
    scale, infinities and NaN."""
    d, block = 64, 16
    q = orc.QMAX[fmt]
    rows = torch.zeros(12 * block, d)
    for i, x in enumerate((0.0, q, math.nextafter(q, 1e9), q * 2.0 ** -120, 1e-44, 3.3895e38, 3.4028e38, 1.0,
                           2.0 ** -126)):
        rows[i * block, 3] = torch.tensor(x, dtype=torch.float64).float()
        rows[i * block + 5, 7] = -rows[i * block, 3] * 0.37
    rows[9 * block + 2] = torch.linspace(-q, q, d)
    rows[10 * block + 1, 5], rows[10 * block + 1, 6], rows[10 * block + 2, 9] = math.inf, -math.inf, 3.0
    rows[11 * block + 1, 5], rows[11 * block + 2, 9] = math.nan, 5.0
    new = [rows[None, None].contiguous(), rows.flip(0)[None, None].contiguous()]
    cache = _cache(1, 1, 12 * block, d, fmt, block, seed=9)
    state = _state(cache)
    _ops().cache_write(cache, new[0].cuda(), new[1].cuda(), pos=0)
    _expect(state, new, [0], [12 * block], block, fmt)
    _same(cache, state, [12 * block], block)
    got = _ops().cache_read(cache, dtype=torch.float32)
    for g, (codes, scale) in zip(got, state):
        want = orc.values(codes, scale, block).float()
        assert torch.equal(g.cpu().isnan(), want.isnan())
        assert torch.equal(g.cpu().nan_to_num(), want.nan_to_num())


def test_write_strided_sources():
    """Token-major sources, sources whose rows are a slice of a wider
    projection, and ones that need a copy (offset base, expanded batch)."""
    ops, b, h, t, d, block = _ops(), 2, 3, 100, 128, 64
    qkv = _rows(b, 1, t, 5 * h * d, torch.bfloat16, 1)[:, 0].cuda()
    wide = qkv.view(b, t, 5 * h, d)
    sources = [wide[:, :, h:2 * h].transpose(1, 2), wide[:, :, 2 * h:3 * h].transpose(1, 2)]
    odd = torch.empty(b * h * t * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(b, h, t, d)
    odd.copy_(sources[0])
    for k, v in (sources, (odd, sources[1]), (sources[0][:1].expand(b, -1, -1, -1), sources[1])):
        cache = _cache(b, h, t, d, "e4m3", block, seed=2)
        state = _state(cache)
        ops.cache_write(cache, k, v, pos=0)
        _expect(state, [k.cpu(), v.cpu()], [0] * b, [t] * b, block, "e4m3")
        _same(cache, state, [t] * b, block)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt,d,block,cap,start,n", [("e4m3", 128, 64, 333, 0, 333), ("int8", 64, 16, 200, 37, 101),
                                                    ("e4m3", 64, 128, 129, 128, 1), ("int8", 128, 32, 64, 5, 0)])
def test_read(fmt, d, block, cap, start, n, dtype):
    b, h = 2, 3
    cache = _cache(b, h, cap, d, fmt, block, pad=1, seed=3)
    new = [_rows(b, h, cap, d, torch.bfloat16, 1 + j) for j in range(2)]
    _ops().cache_write(cache, new[0].cuda(), new[1].cuda(), pos=0)
    got = _ops().cache_read(cache, n_keys=n, start=start, dtype=dtype)
    for g, (codes, scale) in zip(got, _state(cache)):
        want = orc.values(codes, scale, block)[:, :, start:start + n].float().to(dtype)  # exact in fp32
        assert g.dtype == dtype and torch.equal(g.cpu(), want)
    lengths = torch.tensor([start + n // 2, 0], dtype=torch.int32).cuda()
    out = tuple(torch.full((b, h, n, d), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    assert _ops().cache_read(cache, n_keys=n, start=start, dtype=dtype, lengths=lengths, out=out) is out
    for g, w in zip(out, got):
        assert torch.equal(g[0, :, :n // 2], w[0, :, :n // 2])
        assert not g[0, :, n // 2:].any() and not g[1].any()


# ---- attention ------------------------------------------------------------------------------------

def _filled(b, h, cap, d, fmt, block, n, seed=0, pad=0, spread=0.5):
    """A cache whose first n[i] rows of sequence i are written, the rest noise."""
    cache = _cache(b, h, cap, d, fmt, block, pad=pad, seed=seed)
    t = max(max(n), 1)
    new = [_rows(b, h, t, d, torch.bfloat16, seed + 50 + j, spread) for j in range(2)]
    _ops().cache_write(cache, new[0].cuda(), new[1].cuda(), pos=torch.zeros(1, dtype=torch.int32).cuda(),
                       lengths=torch.tensor(n, dtype=torch.int32).cuda(), check=True)
    return cache


def _check_rows(got, q, cache, n, window, sink, sparse, what, scaling=None):
    d = cache.head_dim
    scaling = d ** -0.5 if scaling is None else scaling
    kv = [orc.values(c, s, cache.block) for c, s in _state(cache)]
    for i in range(cache.batch):
        out, spread, slack = orc.attend(q[i, :, 0].float().cpu(), kv[0][i], kv[1][i], n[i], scaling, window, sink,
                                        sparse, (d + 6) * 2.0 ** -23,
                                        1 / 65024 if cache.format == "int8" else 2.0 ** -29)
        vmax = kv[1][i, :, :n[i]].abs().amax().item() if n[i] else 0.0
        tol = 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + n[i] * 2.0 ** -38 * vmax + slack
        err = (got[i, 0].float().cpu().double() - out).abs()
        assert torch.isfinite(got[i].float()).all(), f"{what}: sequence {i} not finite"
        worst = (err / tol.clamp_min(1e-300)).max().item() if n[i] else float(err.max() > 0)
        assert worst <= 1.0, f"{what}: sequence {i} is {worst:.2f} times its tolerance off"


CASES = [
    # fmt, b, H, Hkv, d, block, cap, n, window, sink
    ("e4m3", 1, 32, 8, 128, 64, 2112, [2111], 512, 128),
    ("int8", 2, 8, 1, 128, 32, 1500, [1500, 1500], 300, 7),
    ("e4m3", 3, 4, 4, 64, 16, 777, [777, 1, 0], 100, 3),
    ("int8", 4, 16, 2, 64, 128, 1300, [1299, 17, 300, 64], 256, 0),
    ("e4m3", 1, 2, 1, 128, 64, 64, [1], 1, 0),
    ("e4m3", 2, 6, 2, 128, 16, 400, [400, 399], 0, 33),
    ("int8", 2, 5, 5, 64, 64, 130, [129, 16], 0, 0),
    ("e4m3", 2, 14, 2, 64, 64, 700, [650, 333], 5000, 3),
    ("e4m3", 1, 64, 8, 128, 64, 6000, [5999], 4096, 128),
]


@pytest.mark.parametrize("fmt,b,H,Hkv,d,block,cap,n,window,sink", CASES)
def test_decode(fmt, b, H, Hkv, d, block, cap, n, window, sink):
    ops = _ops()
    cache = _filled(b, Hkv, cap, d, fmt, block, n, seed=cap, pad=1)
    q = _rows(b, H, 1, d, torch.bfloat16, 5).cuda()
    live = torch.tensor(n, dtype=torch.int32).cuda()
    dense, sparse = ops.cache_decode(q, cache, window=window, sink=sink, n_keys_dev=live)
    _check_rows(dense, q, cache, n, window, sink, False, "dense")
    _check_rows(sparse, q, cache, n, window, sink, True, "sparse")
    # one row alone: the sparse row is the same bit for bit (its chunks go by sink and window only)
    alone, none = ops.cache_decode(q, cache, window=window, sink=sink, n_keys_dev=live, want_sparse=False)
    assert none is None
    _check_rows(alone, q, cache, n, window, sink, False, "dense alone")
    alone = ops.cache_decode(q, cache, window=window, sink=sink, n_keys_dev=live, want_dense=False)
    assert alone[0] is None and torch.equal(alone[1], sparse)
    if len(set(n)) == 1:  # a host count
        dense, sparse = ops.cache_decode(q, cache, window=window, sink=sink, n_keys=n[0])
        _check_rows(dense, q, cache, n, window, sink, False, "dense, host count")
        _check_rows(sparse, q, cache, n, window, sink, True, "sparse, host count")
        one = torch.tensor(n[:1], dtype=torch.int32).cuda()
        assert torch.equal(ops.cache_decode(q, cache, window=window, sink=sink, n_keys_dev=one, want_dense=False)[1],
                           ops.cache_decode(q, cache, window=window, sink=sink, n_keys_dev=live, want_dense=False)[1])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300])
def test_decode_every_border(n, fmt):
    """Lengths around groups, blocks and chunks; windows that begin and end
    inside a block."""
    ops = _ops()
    cache = _filled(1, 2, 320, 128, fmt, 16, [n], seed=n)
    q = _rows(1, 8, 1, 128, torch.bfloat16, n).cuda()
    for window, sink in ((16, 0), (n // 2, 5), (33, 1), (1, 16), (0, 1), (0, 0)):
        dense, sparse = ops.cache_decode(q, cache, window=window, sink=sink, n_keys=n)
        _check_rows(dense, q, cache, [n], window, sink, False, f"dense {n}")
        if min(n, window + sink) == 0:
            assert not sparse.any()
        else:
            _check_rows(sparse, q, cache, [n], window, sink, True, f"sparse {n} {window} {sink}")


def test_decode_extreme_scales():
    """Value scales that differ by 2^80 between blocks, keys of all sizes, one
    key that takes all the weight, and a query of subnormal and huge size."""
    ops = _ops()
    b, h, n, d, block = 1, 2, 200, 64, 16
    k, v = _rows(b, h, n, d, torch.float32, 1, 0.3), _rows(b, h, n, d, torch.float32, 2, 0.3)
    v[:, :, 16:32] *= 2.0 ** -70
    v[:, :, 48:64] = 0
    v[:, 1, 64:80] *= 2.0 ** 40
    k[:, :, 80:96] *= 2.0 ** -40
    k[:, 1, 100] *= 60
    cache = _cache(b, h, 208, d, "e4m3", block, seed=3)
    ops.cache_write(cache, k.cuda(), v.cuda(), pos=0)
    for size in (1.0, 30.0, 2.0 ** -125, 2.0 ** 100):
        q = (_rows(b, 4, 1, d, torch.float32, 3, 0.2) * size).to(torch.bfloat16).cuda()
        scaling = d ** -0.5 * (2.0 ** -100 if size > 1e10 else 1.0)
        dense, sparse = ops.cache_decode(q, cache, window=50, sink=9, n_keys=n, scaling=scaling)
        _check_rows(dense, q, cache, [n], 50, 9, False, f"dense {size}", scaling)
        _check_rows(sparse, q, cache, [n], 50, 9, True, f"sparse {size}", scaling)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_decode_keeps_live_nan_visible(fmt, where):
    """A NaN among the live keys or values makes the rows of its heads NaN; one
    outside a key set does not reach that set's row."""
    ops = _ops()
    new = {x: _rows(1, 2, 300, 64, torch.bfloat16, 3 + i) for i, x in enumerate("kv")}
    new[where][0, 1, 40, :] = math.nan
    cache = _cache(1, 2, 320, 64, fmt, 16, seed=8)
    ops.cache_write(cache, new["k"].cuda(), new["v"].cuda(), pos=0)
    q = _rows(1, 4, 1, 64, torch.bfloat16, 6).cuda()
    dense, sparse = ops.cache_decode(q, cache, window=100, sink=10, n_keys=300)
    assert dense[0, 0, 2:].isnan().all() and not dense[0, 0, :2].isnan().any()
    assert not sparse.isnan().any()
    q[0, 0, 0, 0] = math.inf
    dense, _ = ops.cache_decode(q, cache, window=0, sink=0, n_keys=30, want_sparse=False)
    assert dense[0, 0, 0].isnan().all() and not dense[0, 0, 1:].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_decode_other_query_layouts(dtype):
    """Queries of another type are taken as bf16; token-major ones in place."""
    ops = _ops()
    cache = _filled(2, 2, 100, 128, "e4m3", 64, [100, 100], seed=12)
    q = _rows(2, 8, 1, 128, dtype, 4).cuda()
    want = ops.cache_decode(q.to(torch.bfloat16), cache, window=10, sink=1)
    got = ops.cache_decode(q.to(torch.bfloat16).transpose(1, 2).contiguous().transpose(1, 2).to(dtype), cache,
                           window=10, sink=1)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    got = ops.cache_decode(odd, cache, window=10, sink=1)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_decode_long_cache():
    """131072 keys: chunks of the length that a long cache gets, and offsets
    past 32 bits of a cache whose heads lie far apart."""
    ops = _ops()
    n, d = 131072, 128
    cache = _filled(1, 1, n, d, "e4m3", 64, [n], seed=21, spread=0.3)
    q = _rows(1, 4, 1, d, torch.bfloat16, 4).cuda()
    dense, sparse = ops.cache_decode(q, cache, window=2048, sink=128)
    _check_rows(dense, q, cache, [n], 2048, 128, False, "dense")
    _check_rows(sparse, q, cache, [n], 2048, 128, True, "sparse")


def test_offsets_past_32_bits():
    """Two heads whose codes lie more than 2^32 bytes apart."""
    from delta_attention_b200.kv_cache import QuantizedKV, SCALE_TYPE
    ops = _ops()
    n, d = 70, 64
    far = (1 << 32) + 4096
    store = [torch.empty(far + n * d, dtype=torch.int8, device="cuda") for _ in range(2)]
    k, v = (s.as_strided((1, 2, n, d), (2 * far, far, d, 1)) for s in store)
    ks, vs = (torch.zeros(1, 2, 2, dtype=torch.uint8, device="cuda").view(SCALE_TYPE) for _ in range(2))
    cache = QuantizedKV(k, v, ks, vs, 64)
    new = [_rows(1, 2, n, d, torch.bfloat16, 31 + j) for j in range(2)]
    ops.cache_write(cache, new[0].cuda(), new[1].cuda(), pos=0)
    state = [(torch.zeros(1, 2, n, d, dtype=torch.float64), torch.zeros(1, 2, 2, dtype=torch.long)) for _ in range(2)]
    _expect(state, new, [0], [n], 64, "int8")
    _same(cache, state, [n], 64)
    for g, (codes, scale) in zip(ops.cache_read(cache, dtype=torch.float32), state):
        assert torch.equal(g.cpu().double(), orc.values(codes, scale, 64))
    q = _rows(1, 4, 1, d, torch.bfloat16, 4).cuda()
    dense, _ = ops.cache_decode(q, cache, window=0, sink=0, want_sparse=False)
    _check_rows(dense, q, cache, [n], 0, 0, False, "dense")


# ---- streams and graphs ---------------------------------------------------------------------------

def test_step_captured_and_replayed():
    """Write one token and attend, captured once and replayed while the cache
    grows, in two graphs that interleave: every step equals the eager calls."""
    ops = _ops()
    b, H, h, d, block, cap = 2, 8, 2, 64, 16, 200
    fill = [_rows(b, h, 90, d, torch.bfloat16, 1 + j) for j in range(2)]
    toks = [[_rows(b, h, 1, d, torch.bfloat16, 100 + 2 * i + j) * (1 + i % 5) for j in range(2)] for i in range(40)]
    qs = [_rows(b, H, 1, d, torch.bfloat16, 500 + i).cuda() for i in range(40)]
    caches = [_cache(b, h, cap, d, "e4m3", block, seed=5) for _ in range(2)]
    for c in caches:
        ops.cache_write(c, fill[0].cuda(), fill[1].cuda(), pos=0)
    kt, vt = (torch.zeros(b, h, 1, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qt = torch.zeros_like(qs[0])
    pos = torch.full((b,), 90, dtype=torch.int32, device="cuda")
    n = pos + 1

    def step():
        ops.cache_write(caches[1], kt, vt, pos=pos)
        return ops.cache_decode(qt, caches[1], window=40, sink=4, n_keys_dev=n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(40):
        kt.copy_(toks[i][0])
        vt.copy_(toks[i][1])
        qt.copy_(qs[i])
        pos.fill_(90 + i)
        n.fill_(91 + i)
        graphs[i % 2].replay()
        ops.cache_write(caches[0], toks[i][0].cuda(), toks[i][1].cuda(), pos=90 + i)
        want = ops.cache_decode(qs[i], caches[0], window=40, sink=4, n_keys_dev=n)
        assert torch.equal(outs[i % 2][0], want[0]) and torch.equal(outs[i % 2][1], want[1]), i
    ops.check_errors()


def test_first_calls_within_a_capture():
    """A process whose first calls of these kernels are captured (no eager run
    before): the replays do what the eager calls then do."""
    import subprocess
    import sys
    code = """
import torch
from delta_attention_b200 import ops
from delta_attention_b200.kv_cache import QuantizedKV
caches = [QuantizedKV.allocate(1, 2, n, 64, format=f, block=16) for n, f in ((6000, 'e4m3'), (300, 'int8'))]
g = torch.Generator(device='cuda').manual_seed(0)
k, v = (torch.randn(1, 2, 300, 64, generator=g, device='cuda') for _ in range(2))
q = torch.randn(1, 8, 1, 64, generator=g, device='cuda').bfloat16()
live = torch.tensor([300], dtype=torch.int32, device='cuda')
def step():
    out = []
    for c in caches:
        ops.cache_write(c, k, v, pos=0)
        out += ops.cache_decode(q, c, window=100, sink=9, n_keys_dev=live)
        out += ops.cache_read(c, n_keys=300)
    return out
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
for x, y in zip(got, step()):
    assert x.abs().sum() > 0 and torch.equal(x, y)
ops.check_errors()
print('same')
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


def test_calls_on_two_streams():
    """Calls on two streams at once do not share a workspace, and repeat bit for bit."""
    ops = _ops()
    cache = _filled(2, 4, 3000, 128, "int8", 64, [3000, 2900], seed=15)
    live = torch.tensor([3000, 2900], dtype=torch.int32).cuda()
    qs = [_rows(2, 16, 1, 128, torch.bfloat16, i).cuda() for i in range(2)]
    want = [ops.cache_decode(q, cache, window=500, sink=64, n_keys_dev=live) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.cache_decode(qs[i], cache, window=500, sink=64, n_keys_dev=live))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x[0], want[i][0]) and torch.equal(x[1], want[i][1])


def test_calls_from_another_current_device(monkeypatch):
    """Where the cache's device is not the current one, an op runs again with it
    current (here the check is made to say so once)."""
    ops = _ops()
    cache = _filled(1, 2, 100, 64, "e4m3", 64, [100], seed=12)
    q = _rows(1, 4, 1, 64, torch.bfloat16, 4).cuda()
    x = _rows(1, 2, 3, 64, torch.bfloat16, 4).cuda()
    entered = []

    def once(answers):
        left = list(answers)
        monkeypatch.setattr(ops, "_is_current", lambda c: left.pop(0))

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    want = ops.cache_decode(q, cache, window=10, sink=1)
    monkeypatch.setattr(torch.cuda, "device", Device)
    once([False, True])
    got = ops.cache_decode(q, cache, window=10, sink=1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    once([False, True])
    ops.cache_write(cache, x, x, pos=97)
    once([False, True])
    k, _ = ops.cache_read(cache, n_keys=3, start=97, dtype=torch.float32)
    assert k.abs().sum() > 0 and entered == [0, 0, 0]


def test_calls_of_two_threads_on_one_stream():
    """Two host threads that decode on the same stream: each call's launches
    stay together, so the shared workspace holds one call's partials at a time."""
    import threading
    ops = _ops()
    cache = _filled(1, 8, 20000, 64, "e4m3", 64, [20000], seed=16)  # (long enough for a merge launch)
    qs = [_rows(1, 16, 1, 64, torch.bfloat16, i).cuda() for i in range(2)]
    want = [ops.cache_decode(q, cache, window=500, sink=64) for q in qs]
    got, stream = [[], []], torch.cuda.Stream()
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(stream):
            for _ in range(50):
                got[i].append(ops.cache_decode(qs[i], cache, window=500, sink=64))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 50
        for x in got[i]:
            assert torch.equal(x[0], want[i][0]) and torch.equal(x[1], want[i][1])


def test_no_keys_at_all():
    """A host count of zero, and reads and writes of nothing."""
    ops = _ops()
    cache = _cache(2, 2, 100, 64, "e4m3", 16, seed=1)
    before = _raw(cache)
    dense, sparse = ops.cache_decode(_rows(2, 4, 1, 64, torch.bfloat16, 1).cuda(), cache, window=10, sink=2, n_keys=0)
    assert not dense.any() and not sparse.any()
    empty = torch.empty(2, 2, 0, 64, dtype=torch.bfloat16, device="cuda")
    ops.cache_write(cache, empty, empty, pos=100, check=True)
    k, v = ops.cache_read(cache, n_keys=0, start=100)
    assert tuple(k.shape) == tuple(v.shape) == (2, 2, 0, 64)
    assert all(torch.equal(x, y) for x, y in zip(before, _raw(cache)))


def test_ops_refuse_mismatched_tensors():
    """Refused before any launch: the cache and the outputs are not touched."""
    ops = _ops()
    cache = _cache(2, 2, 100, 64, "int8", 16, seed=1)
    x = _rows(2, 2, 3, 64, torch.bfloat16, 1).cuda()
    q = _rows(2, 4, 1, 64, torch.bfloat16, 1).cuda()
    n = torch.tensor([3, 3], dtype=torch.int32).cuda()
    for call in (lambda: ops.cache_write(cache, x[:1], x[:1], pos=0),
                 lambda: ops.cache_write(cache, x, x[:, :, :2], pos=0),
                 lambda: ops.cache_write(cache, x, x.half(), pos=0),
                 lambda: ops.cache_write(cache, x.int(), x.int(), pos=0),
                 lambda: ops.cache_write(cache, x, x, pos=98), lambda: ops.cache_write(cache, x, x, pos=-1),
                 lambda: ops.cache_write(cache, x.cpu(), x.cpu(), pos=0),
                 lambda: ops.cache_write(cache, x, x, pos=n.long()), lambda: ops.cache_write(cache, x, x, pos=n.cpu()),
                 lambda: ops.cache_write(cache, x, x, pos=0, lengths=n.repeat(2)),
                 lambda: ops.cache_read(cache, n_keys=101), lambda: ops.cache_read(cache, start=-1),
                 lambda: ops.cache_read(cache, dtype=torch.float64), lambda: ops.cache_read(cache, out=(x, x)),
                 lambda: ops.cache_decode(q[:1], cache, window=1, sink=1),
                 lambda: ops.cache_decode(q.expand(2, 4, 2, 64), cache, window=1, sink=1),
                 lambda: ops.cache_decode(q.cpu(), cache, window=1, sink=1),
                 lambda: ops.cache_decode(q, cache, window=1, sink=1, n_keys=101),
                 lambda: ops.cache_decode(q, cache, window=1, sink=1, n_keys_dev=n.float()),
                 lambda: ops.cache_decode(q, cache, window=1, sink=1, want_dense=False, want_sparse=False)):
        with pytest.raises(ValueError):
            call()
    from delta_attention_b200._lib import DtaError
    for heads in (3, 18):  # not a multiple of the KV heads; more than 8 to one
        with pytest.raises(DtaError, match="SHAPE"):
            ops.cache_decode(_rows(2, heads, 1, 64, torch.bfloat16, 1).cuda(), cache, window=1, sink=1)


@pytest.mark.parametrize("far", [101, 2 ** 31, 2 ** 32 + 5])
def test_window_and_sink_beyond_the_cache(far):
    """More than the cache holds means all keys, past 32 bits too; a negative one is refused."""
    ops = _ops()
    cache = _cache(1, 2, 100, 64, "e4m3", 32, seed=8)
    x = _rows(1, 2, 100, 64, torch.bfloat16, 9).cuda()
    ops.cache_write(cache, x, x, pos=0)
    q = _rows(1, 4, 1, 64, torch.bfloat16, 10).cuda()
    for kw in (dict(window=far, sink=0), dict(window=0, sink=far), dict(window=far, sink=far)):
        _, sparse = ops.cache_decode(q, cache, want_dense=False, **kw)
        _check_rows(sparse, q, cache, [100], kw["window"], kw["sink"], True, f"{kw}")
    for kw in (dict(window=-far, sink=0), dict(window=0, sink=-far)):
        with pytest.raises(ValueError, match="negative"):
            ops.cache_decode(q, cache, **kw)


def test_write_read_attend_together():
    """A prompt in chunks, then single tokens, as a decode loop runs them: the
    attention over the cache equals the dense path over what reads back, and
    the rows kernel over the read-back prefix continues a prompt."""
    ops = _ops()
    b, H, h, d, block = 1, 8, 2, 128, 64
    k, v = (_rows(b, h, 700, d, torch.bfloat16, 60 + j, 0.3) for j in range(2))
    cache = _cache(b, h, 768, d, "e4m3", block, seed=6)
    at = 0
    for t in (300, 129, 64, 1, 1, 1, 200, 4):
        ops.cache_write(cache, k[:, :, at:at + t].cuda(), v[:, :, at:at + t].cuda(), pos=at)
        at += t
    assert at == 700
    q = _rows(b, H, 8, d, torch.bfloat16, 70, 0.3).cuda()
    kr, vr = ops.cache_read(cache, n_keys=at)
    rows = torch.arange(8, dtype=torch.int32)
    out = ops.rows(q, kr, vr, rows, rows + at - 8)
    last = q[:, :, 7:].contiguous()
    got, _ = ops.cache_decode(last, cache, window=0, sink=0, n_keys=at, want_sparse=False)
    ref, _ = ops.decode(last, kr, vr, window=0, sink=0, want_sparse=False)
    _check_rows(got, last, cache, [at], 0, 0, False, "dense")
    # the bf16 kernels round their weights to bf16 (2^-8 of W where fp16 has 2^-11)
    kv = [orc.values(c, s, block)[0] for c, s in _state(cache)]
    o, w, _ = orc.attend(last[0, :, 0].float().cpu(), kv[0], kv[1], at, d ** -0.5, 0, 0, False)
    tol = (2.0 ** -7 * o.abs() + 2.0 ** -6 * w)
    for x in (ref[0, 0], out[0, 7]):
        assert ((x.float().cpu().double() - got[0, 0].float().cpu().double()).abs() <= tol).all()
