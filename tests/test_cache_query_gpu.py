"""The 8-bit cache's attention with queries that have a strong channel."""

import pytest
import torch

from tests._cache_check import check_rows

pytestmark = pytest.mark.gpu


def _attend(q, cache, n, window, sink, scaling=None):
    from delta_attention_b200 import ops
    dense, sparse = ops.cache_decode(q, cache, window=window, sink=sink, n_keys=n, scaling=scaling)
    check_rows(dense, q, cache, [n] * cache.batch, window, sink, False, "dense", scaling)
    check_rows(sparse, q, cache, [n] * cache.batch, window, sink, True, "sparse", scaling)


@pytest.mark.parametrize("size", [1.0, 200.0, 5000.0])
@pytest.mark.parametrize("fmt,d,H,Hkv", [("int8", 128, 8, 2), ("int8", 64, 8, 1), ("int8", 128, 3, 3), ("e4m3", 128, 8, 2),
                                         ("e4m3", 64, 8, 1)])
def test_query_with_a_strong_channel(fmt, d, H, Hkv, size):
    """One channel of the query is ``size`` times the others, and the keys are zero there: the other channels
    alone decide the weights, and keep the bits that bf16 gave them."""
    from delta_attention_b200 import ops
    from delta_attention_b200.kv_cache import QuantizedKV
    g = torch.Generator().manual_seed(d + H)
    n = 41
    k, v = torch.randn(2, Hkv, n, d, generator=g), torch.randn(2, Hkv, n, d, generator=g)
    q = torch.randn(2, H, 1, d, generator=g)
    k[..., 7] = 0
    q[..., 7] = 1.5 * size
    cache = QuantizedKV.allocate(2, Hkv, 64, d, format=fmt, block=16)
    ops.cache_write(cache, k.cuda(), v.cuda(), pos=0)
    _attend(q.to(torch.bfloat16).cuda(), cache, n, 17, 3)
