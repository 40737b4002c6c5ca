"""The 8-bit cache's attention with block scales far apart, each row held to what its own
keys and values allow (zeros in a row's place do not pass)."""

import pytest
import torch

from tests._cache_check import check_rows

pytestmark = pytest.mark.gpu

BLOCK, N, D = 16, 200, 64


def inputs():
    """K, V [1, 2, N, D]: values of one block 2^-70 times the others', of another zero, of a third 2^40 times
    them in one head; a block of small keys, and one key that takes most of the weight."""
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(1, 2, N, D, generator=g), torch.randn(1, 2, N, D, generator=g)
    v[:, :, 16:32] *= 2.0 ** -70
    v[:, :, 48:64] = 0
    v[:, 1, 64:80] *= 2.0 ** 40
    k[:, :, 80:96] *= 2.0 ** -40
    k[:, 1, 100] *= 60
    return k, v


def query(size):
    q = torch.randn(1, 4, 1, D, generator=torch.Generator().manual_seed(3))
    return (q * size).to(torch.bfloat16), D ** -0.5 * (2.0 ** -100 if size > 1e10 else 1.0)


SIZES = (1.0, 30.0, 2.0 ** -125, 2.0 ** 100)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scales_far_apart(fmt, size):
    from delta_attention_b200 import ops
    from delta_attention_b200.kv_cache import QuantizedKV
    cache = QuantizedKV.allocate(1, 2, 208, D, format=fmt, block=BLOCK)
    ops.cache_write(cache, *(x.cuda() for x in inputs()), pos=0)
    q, scaling = query(size)
    q = q.cuda()
    for window, sink in ((50, 9), (130, 0), (5, 25), (0, 70)):
        dense, sparse = ops.cache_decode(q, cache, window=window, sink=sink, n_keys=N, scaling=scaling)
        check_rows(dense, q, cache, [N], window, sink, False, f"dense {size}", scaling)
        check_rows(sparse, q, cache, [N], window, sink, True, f"sparse {size} {window} {sink}", scaling)
    live = torch.tensor([N], dtype=torch.int32).cuda()
    for n in (17, 31, 64, 80):  # rows that end within and behind the odd blocks
        dense, _ = ops.cache_decode(q, cache, window=0, sink=0, n_keys_dev=live.fill_(n), want_sparse=False,
                                    scaling=scaling)
        check_rows(dense, q, cache, [n], 0, 0, False, f"dense {size} {n}", scaling)
