"""8-bit KV cache without a GPU: the handle's checks, the C ABI's refusals (all
before any CUDA call), and the oracle against torch's own conversions."""

import ctypes

import pytest
import torch

from delta_attention_b200 import _lib, ops
from delta_attention_b200.kv_cache import SCALE_TYPE, QuantizedKV
from oracle import cache_oracle as orc

FAKE = 1 << 20  # never dereferenced: validation fails before any CUDA call


def _tensors(b=2, h=3, cap=100, d=64, block=16, dtype=torch.int8):
    k = torch.zeros(b, h, cap, d, dtype=torch.uint8).view(dtype)
    s = torch.zeros(b, h, -(-cap // block), dtype=torch.uint8).view(SCALE_TYPE)
    return dict(k=k, v=k.clone(), k_scale=s, v_scale=s.clone(), block=block)


def test_handle_describes_its_tensors():
    t = _tensors(dtype=torch.float8_e4m3fn)
    c = QuantizedKV(**t)
    assert (c.batch, c.n_kv_heads, c.capacity, c.head_dim, c.format, c.block) == (2, 3, 100, 64, "e4m3", 16)
    d = c._decode_args.cache
    assert (d.k, d.v_scale) == (t["k"].data_ptr(), t["v_scale"].data_ptr())
    assert (d.k_stride_b, d.k_stride_h, d.k_stride_s) == (3 * 100 * 64, 100 * 64, 64)
    assert (d.k_scale_stride_b, d.k_scale_stride_h) == (21, 7)
    a = QuantizedKV.allocate(1, 2, 70, 128, format="int8", block=64, device="cpu")
    assert a.k.dtype == torch.int8 and tuple(a.k_scale.shape) == (1, 2, 2) and a.nbytes() == 2 * (2 * 70 * 128 + 4)


@pytest.mark.parametrize("change,match", [
    (dict(block=48), "block"),
    (dict(k=torch.zeros(2, 3, 100, 64)), "float8_e4m3fn or int8"),
    (dict(v=torch.zeros(2, 3, 100, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)), "float8_e4m3fn or int8"),
    (dict(v=torch.zeros(2, 3, 99, 64, dtype=torch.int8)), "codes must be two"),
    (dict(k_scale=torch.zeros(2, 3, 7)), "k_scale"),
    (dict(v_scale=torch.zeros(2, 3, 6, dtype=torch.uint8).view(SCALE_TYPE)), "v_scale"),
    (dict(k_scale=torch.zeros(2, 7, 3, dtype=torch.uint8).view(SCALE_TYPE).transpose(1, 2)), "contiguous blocks"),
    (dict(k=torch.zeros(2, 3, 64, 100, dtype=torch.int8).transpose(2, 3)), "d contiguous"),
    (dict(k=torch.zeros(2, 3, 100, 72, dtype=torch.int8)[..., :64]), "16 bytes"),
    (dict(k=torch.zeros(1, 3, 100, 64, dtype=torch.int8).expand(2, -1, -1, -1)), "16 bytes"),
    (dict(k=torch.zeros(2 * 3 * 100 * 64 + 8, dtype=torch.int8)[8:].view(2, 3, 100, 64)), "16 bytes"),
])
def test_handle_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        QuantizedKV(**{**_tensors(), **change})


def test_handle_refuses_sizes():
    with pytest.raises(ValueError, match="head_dim"):
        QuantizedKV(**_tensors(d=96))
    with pytest.raises(ValueError, match="empty"):
        QuantizedKV(**_tensors(cap=0))
    with pytest.raises(ValueError, match="format"):
        QuantizedKV.allocate(1, 1, 16, 64, format="fp4", device="cpu")
    with pytest.raises(ValueError, match="block"):
        QuantizedKV.allocate(1, 1, 16, 64, block=0, device="cpu")


def test_ops_refuse_cpu_tensors():
    c = QuantizedKV(**_tensors())
    x = torch.zeros(2, 3, 1, 64)
    for call in (lambda: ops.cache_write(c, x, x, pos=0), lambda: ops.cache_read(c),
                 lambda: ops.cache_decode(x, c, window=1, sink=1), lambda: ops.cache_read(cache=c)):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call()


def _args(kind):
    a = kind()
    a.abi_version = _lib.ABI_VERSION
    c = a.cache
    c.batch, c.n_kv_heads, c.capacity, c.head_dim, c.block, c.format = 2, 4, 1000, 128, 64, 0
    c.k = c.v = c.k_scale = c.v_scale = FAKE
    c.k_stride_b, c.k_stride_h, c.k_stride_s = 4 * 128000, 128000, 128
    c.v_stride_b, c.v_stride_h, c.v_stride_s = 4 * 128000, 128000, 128
    c.k_scale_stride_b, c.k_scale_stride_h, c.v_scale_stride_b, c.v_scale_stride_h = 64, 16, 64, 16
    if kind is _lib.CacheWriteArgs:
        a.n_new, a.pos, a.k_new, a.v_new = 5, 3, FAKE, FAKE
        for x in "kv":
            for s, n in zip("bhs", (2560, 640, 128)):
                setattr(a, f"{x}_new_stride_{s}", n)
    elif kind is _lib.CacheReadArgs:
        a.n_keys, a.out_k, a.out_v = 7, FAKE, FAKE
    else:
        a.n_heads, a.n_keys, a.window, a.sink, a.scaling = 8, 900, 64, 4, 0.1
        a.q = a.dense_out = a.sparse_out = FAKE
        a.q_stride_b, a.q_stride_h = 1024, 128
    return a


def _call(a):
    L = _lib.lib()
    f = {_lib.CacheWriteArgs: L.dta_cache_write, _lib.CacheReadArgs: L.dta_cache_read,
         _lib.CacheDecodeArgs: L.dta_cache_decode}[type(a)]
    return f(ctypes.byref(a), None)


@pytest.mark.parametrize("kind", [_lib.CacheWriteArgs, _lib.CacheReadArgs, _lib.CacheDecodeArgs])
@pytest.mark.parametrize("field,value,status", [
    ("batch", 0, 2), ("n_kv_heads", -1, 2), ("capacity", 0, 2), ("capacity", (1 << 30) + 1, 2), ("head_dim", 96, 6),
    ("block", 48, 1), ("block", 8, 1), ("format", 2, 1), ("k", None, 1), ("v_scale", None, 1), ("v", FAKE + 8, 4),
    ("k_stride_s", 120, 3), ("v_stride_b", 0, 3), ("k_scale_stride_h", 0, 3), ("batch", 20000, 2),
])
def test_abi_refuses_caches(kind, field, value, status):
    a = _args(kind)
    setattr(a.cache, field, value)
    assert _call(a) == status


@pytest.mark.parametrize("kind,change,status", [
    (_lib.CacheWriteArgs, dict(abi_version=99), 1),
    (_lib.CacheWriteArgs, dict(n_new=-1), 2),
    (_lib.CacheWriteArgs, dict(n_new=1001, pos=0), 2),
    (_lib.CacheWriteArgs, dict(pos=-1), 2),
    (_lib.CacheWriteArgs, dict(pos=996), 2),
    (_lib.CacheWriteArgs, dict(src_type=3), 1),
    (_lib.CacheWriteArgs, dict(k_new=None), 1),
    (_lib.CacheWriteArgs, dict(v_new=FAKE + 2), 4),
    (_lib.CacheWriteArgs, dict(k_new_stride_s=124), 3),
    (_lib.CacheWriteArgs, dict(pos_dev=FAKE, n_pos=3), 2),
    (_lib.CacheWriteArgs, dict(pos_dev=FAKE + 2, n_pos=1), 4),
    (_lib.CacheWriteArgs, dict(lengths=FAKE, n_lengths=0), 2),
    (_lib.CacheWriteArgs, dict(error_word=FAKE + 1), 4),
    (_lib.CacheWriteArgs, dict(n_new=0), 0),
    (_lib.CacheReadArgs, dict(abi_version=2), 1),
    (_lib.CacheReadArgs, dict(start=-1), 2),
    (_lib.CacheReadArgs, dict(start=994), 2),
    (_lib.CacheReadArgs, dict(n_keys=-1), 2),
    (_lib.CacheReadArgs, dict(dst_type=-1), 1),
    (_lib.CacheReadArgs, dict(out_k=None), 1),
    (_lib.CacheReadArgs, dict(out_v=FAKE + 8), 4),
    (_lib.CacheReadArgs, dict(lengths=FAKE, n_lengths=4), 2),
    (_lib.CacheReadArgs, dict(start=1000, n_keys=0), 0),
    (_lib.CacheDecodeArgs, dict(abi_version=0), 1),
    (_lib.CacheDecodeArgs, dict(n_heads=10), 2),
    (_lib.CacheDecodeArgs, dict(n_heads=64), 2),
    (_lib.CacheDecodeArgs, dict(n_keys=1001), 2),
    (_lib.CacheDecodeArgs, dict(n_keys=-1), 2),
    (_lib.CacheDecodeArgs, dict(window=-1), 1),
    (_lib.CacheDecodeArgs, dict(q=None), 1),
    (_lib.CacheDecodeArgs, dict(dense_out=None, sparse_out=None), 1),
    (_lib.CacheDecodeArgs, dict(q=FAKE + 4), 4),
    (_lib.CacheDecodeArgs, dict(sparse_out=FAKE + 4), 4),
    (_lib.CacheDecodeArgs, dict(q_stride_h=100), 3),
    (_lib.CacheDecodeArgs, dict(n_keys_dev=FAKE, n_lengths=3), 2),
    (_lib.CacheDecodeArgs, dict(), 7),
    (_lib.CacheDecodeArgs, dict(workspace=FAKE, workspace_bytes=100), 7),
])
def test_abi_refuses_calls(kind, change, status):
    a = _args(kind)
    for k, v in change.items():
        setattr(a, k, v)
    assert _call(a) == status


def test_decode_workspace_size():
    """Never less for more keys, and bounded however long the cache is."""
    L = _lib.lib()
    a = _args(_lib.CacheDecodeArgs)
    a.cache.capacity = 1 << 30
    for window, sink in ((64, 4), (0, 0), (1030, 128), (5000, 33), (1 << 30, 1 << 30)):
        a.window, a.sink, last = window, sink, 0
        for n in [*range(0, 3000, 37), 5000, 10000, 100000, 1 << 20, 1 << 25, 1 << 30]:
            a.n_keys = n
            size = L.dta_cache_decode_workspace_size(ctypes.byref(a))
            assert size >= max(last, 1), (window, sink, n)
            last = size
        assert last <= (8 * 160 * 2 + 8 * 2050) * 2 * 132 * 4 + 512
    a.cache.block = 7
    assert L.dta_cache_decode_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("batch,heads,d", [(1, 8, 128), (641, 1, 64), (643, 5, 128), (1283, 3, 64), (2001, 1, 128)])
def test_decode_workspace_holds_empty_partials(batch, heads, d):
    """Without keys each set still writes one partial per query head: 4 + d
    words, the second set's behind the first's, rounded up to 256 bytes."""
    L = _lib.lib()
    a = _args(_lib.CacheDecodeArgs)
    a.cache.batch, a.cache.n_kv_heads, a.cache.head_dim = batch, 1, d
    a.n_heads, a.n_keys, a.window, a.sink = heads, 0, 0, 0
    one = batch * heads * (4 + d) * 4
    assert L.dta_cache_decode_workspace_size(ctypes.byref(a)) >= -(-one // 256) * 256 + one


# ---- the oracle itself ------------------------------------------------------------------------------

def test_oracle_rounding_is_torchs():
    x = torch.cat((torch.linspace(-448, 448, 40001), torch.linspace(-0.07, 0.07, 40001),
                   torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(0.0)))
    assert torch.equal(orc.round_code(x, "e4m3"), x.to(torch.float8_e4m3fn).double())
    y = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.49])
    assert orc.round_code(y, "int8").tolist() == [0, 2, 2, 0, -2, 126, -126]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_scale_is_the_least(fmt):
    q = orc.QMAX[fmt]
    for amax in (q, q * 1.0000001, q * 0.9999999, 1.0, 3e38, 2.0 ** -100, q * 2.0 ** -126, 1e-44, 0.0):
        u = orc.need(amax, fmt)
        assert u == 1 or amax > q * 2.0 ** (u - 128)
        assert amax <= q * 2.0 ** (u - 127)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_appending_stays_within_one_rounding(fmt):
    """Token by token or at once: the values differ by less than one step of
    the block's final scale (e4m3: only below the normal range)."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 64, generator=g) * torch.exp(torch.linspace(-3, 3, 64))[:, None]
    once, step = torch.zeros(64, 64, dtype=torch.float64), torch.zeros(64, 64, dtype=torch.float64)
    s1, s2 = torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long)
    orc.write_rows(once, s1, x, 0, 64, fmt)
    for i in range(64):
        orc.write_rows(step, s2, x[i:i + 1], i, 64, fmt)
    assert torch.equal(s1, s2)
    if fmt == "int8":
        assert (once - step).abs().max() <= 1
    else:
        normal = once.abs() >= 2.0 ** -6
        assert torch.equal(once[normal], step[normal]) and (once - step).abs().max() <= 2.0 ** -9
    err = (orc.values(step[None], s2[None], 64)[0] - x.double()).abs()
    scale = 2.0 ** (int(s2[0]) - 127)
    most = scale if fmt == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, torch.tensor(scale * 2.0 ** -9))
    assert (err <= most).all()
