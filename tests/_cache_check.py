"""Checks of ``cache_decode`` rows against the 64-bit oracle, with what a row may be off by
taken from the row's own keys and values.

Per output element, with weights w over the row's key set, W = sum w |v|,
off_j = scaling * (c |q| . |k_j| + e max|q| sum|k_j|), s_j the scores in base 2, 2^e_j
the value scales and V_j the value codes:
  2^-8 |out|               the output's rounding to bf16 (half a step)
  2^-11 W                  the weights' rounding to fp16
  2^-39 2^(r - m) sum|V_j| / l   weights below fp16's normal range: half a step is 2^-25 of the factor 2^14 at
                           the largest s_j + e_j = r; m = max s_j, l = sum 2^(s_j - m)
  sum w off |v| + (sum w off) W   the scores, off by off_j.  c = (d + 6) 2^-23: sums over d terms in fp32 (d
                           steps, and 6 more for the products with the scales and log2 e).  e: the query's
                           rounding, 2^-29 for e4m3 and QUERY_STEP for int8
  2^-13 W                  sums of weights and products in fp32, exp2, the maxima's shifts
NaN has to be where the oracle has it, element by element.
"""

import math

import torch

from oracle import cache_oracle as orc

QUERY_STEP = {"e4m3": 2.0 ** -29, "int8": 2.0 ** -23}


def state(cache):
    """[(codes float64, scale bytes int64)] of K and V on the CPU."""
    return [(c.float().cpu().double(), s.view(torch.uint8).cpu().long())
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


def expected(q, kv, block, fmt, n, scaling, window, sink, sparse):
    """One sequence: q [H, d], kv :func:`state` of its heads.  Returns (out, tolerance) [H, d]."""
    (kc, ku), (vc, vu) = kv
    H, d = q.shape
    group = H // kc.shape[0]
    k, v = orc.values(kc, ku, block), orc.values(vc, vu, block)
    out, spread, slack = orc.attend(q, k, v, n, scaling, window, sink, sparse, (d + 6) * 2.0 ** -23, QUERY_STEP[fmt])
    floor = torch.zeros_like(out)
    keys = orc.key_set(n, window, sink, sparse)
    for h in range(H) if len(keys) else ():
        s = k[h // group, keys] @ q[h].double() * (scaling * math.log2(math.e))
        e = vu[h // group, keys // block].double() - 127
        e = torch.where(e == 128, -math.inf, e)  # (a block that reads as NaN)
        m, r = s.max(), (s + e).max()
        floor[h] = 2.0 ** -39 * torch.exp2(r - m) / torch.exp2(s - m).sum() * vc[h // group, keys].abs().sum(dim=0)
    return out, 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + slack + floor


def check_rows(got, q, cache, n, window, sink, sparse, what, scaling=None, blind=False):
    """``got`` [b, 1, H, d] is the row of the key set.  Unless ``blind``, zeros in place of a head's row
    would not pass."""
    scaling = cache.head_dim ** -0.5 if scaling is None else scaling
    kv = state(cache)
    for i in range(cache.batch):
        out, tol = expected(q[i, :, 0].float().cpu(), [(c[i], u[i]) for c, u in kv], cache.block, cache.format, n[i],
                            scaling, window, sink, sparse)
        row = got[i, 0].float().cpu().double()
        assert torch.equal(row.isnan(), out.isnan()), \
            f"{what}: sequence {i} has {int(row.isnan().sum())} NaN where {int(out.isnan().sum())} are due"
        live = ~out.isnan()
        worst = ((row - out).abs() / tol.clamp_min(1e-300))[live].max().item() if live.any() else 0.0
        assert worst <= 1.0, f"{what}: sequence {i} is {worst:.2f} times its tolerance off"
        if not blind:
            assert ((out.abs() > tol) | ~live).any(dim=1).all(), f"{what}: zeros would pass in sequence {i}"
