"""A NaN among the live keys or values of an 8-bit cache is seen in the rows that attend it,
whichever chunk of the key set holds it and however small that chunk's weight is."""

import math

import pytest
import torch

from tests._cache_check import check_rows

pytestmark = pytest.mark.gpu


def _fill(fmt, d, block, n, rows, where, steep=None):
    """Two sequences of n keys and two KV heads; element 5 of ``rows`` of K or V of the
    first sequence's second head is NaN.  ``steep`` = (q, keys): those keys' scores lie
    some 800 binary orders below the others'."""
    from delta_attention_b200 import ops
    from delta_attention_b200.kv_cache import QuantizedKV
    g = torch.Generator().manual_seed(n + d + block)
    new = {x: torch.randn(2, 2, n, d, generator=g) for x in "kv"}
    if steep is not None:
        q, far = steep
        new["k"] = 0.1 * new["k"] + 2 * q[:, ::4].float().cpu()
        new["k"][:, :, far] -= 4 * q[:, ::4].float().cpu()
    new[where][0, 1, rows, 5] = math.nan
    cache = QuantizedKV.allocate(2, 2, n + 40, d, format=fmt, block=block)
    ops.cache_write(cache, new["k"].cuda(), new["v"].cuda(), pos=0)
    return cache


def _attend_every_way(q, cache, n, window, sink, scaling=None):
    """Both rows in clusters (a host count), both with a merge launch (counts of each
    sequence), and each row alone."""
    from delta_attention_b200 import ops
    kw = dict(window=window, sink=sink, scaling=scaling)
    live = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    for what, count in (("host count", dict(n_keys=n)), ("device counts", dict(n_keys_dev=live))):
        for dense, sparse in ((True, True), (True, False), (False, True)):
            rows = ops.cache_decode(q, cache, want_dense=dense, want_sparse=sparse, **count, **kw)
            for row, is_sparse in zip(rows, (False, True)):
                if row is not None:
                    check_rows(row, q, cache, [n, n], window, sink, is_sparse,
                               f"{'sparse' if is_sparse else 'dense'} {what} {dense}{sparse}", scaling)


def _queries(d):
    return torch.randn(2, 8, 1, d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16).cuda()


# rows with a NaN, and the key count: the first token, whose block covers the sink's chunk; one in every block of
# the first 256 keys, which are whole chunks of a dense row; the newest token, alone in the last chunk
PLACES = {"sink": ([0], 300), "first keys": (list(range(3, 256, 16)), 300), "newest": ([256], 257)}


@pytest.mark.parametrize("where", ["v", "k"])
@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("fmt,d,block", [("int8", 128, 128), ("int8", 128, 64), ("int8", 64, 128), ("int8", 64, 64),
                                         ("int8", 64, 16), ("e4m3", 128, 64), ("e4m3", 64, 128)])
def test_nan_reaches_every_row_that_attends_it(fmt, d, block, place, where):
    rows, n = PLACES[place]
    cache = _fill(fmt, d, block, n, rows, where)
    _attend_every_way(_queries(d), cache, n, 64, 4)


@pytest.mark.parametrize("fmt,d", [("e4m3", 128), ("e4m3", 64), ("int8", 128), ("int8", 64)])
def test_nan_of_a_chunk_without_weight_is_kept(fmt, d):
    """Keys whose weights are zero in any arithmetic: zero times NaN is NaN."""
    n, q = 300, _queries(d)
    # one query per KV head that its keys follow (queries 0 and 4), the others as they come
    cache = _fill(fmt, d, 64, n, [1, 70], "v", (q, slice(0, 256)))
    _attend_every_way(q, cache, n, 20, 100, scaling=1.0)


@pytest.mark.parametrize("fmt,n", [("int8", 40000), ("e4m3", 40000)])
def test_nan_of_one_chunk_among_many(fmt, n):
    """More chunks than one round of the merge takes: the NaN in the first of them."""
    cache = _fill(fmt, 128, 128, n, list(range(0, 1024, 128)), "v")
    _attend_every_way(_queries(128), cache, n, 2048, 128)
