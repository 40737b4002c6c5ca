"""CPU oracle of the 8-bit KV cache, in 64 bits and from its definition.

Codes of a block with scale byte u stand for code * 2^(u - 127).  Tensors here
hold the codes' values as float64 and the scale bytes as int64.
"""

from __future__ import annotations

import math

import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}


def round_code(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """Nearest value of the format, ties to even (|x| <= qmax; NaN stays)."""
    x = x.double()
    if fmt == "int8":
        return torch.round(x)
    mag = torch.nan_to_num(x).abs().clamp_min(2.0 ** -60)
    step = torch.exp2(torch.floor(torch.log2(mag)).clamp_min(-6.0) - 3)
    return torch.round(x / step) * step


def need(amax: float, fmt: str) -> int:
    """Smallest u >= 1 with amax <= qmax * 2^(u - 127)."""
    if amax == 0:
        return 1
    u = max(1, 127 + math.floor(math.log2(amax)) - 10)
    while amax > QMAX[fmt] * 2.0 ** (u - 127):
        u += 1
    return u


def write_rows(codes: torch.Tensor, scale: torch.Tensor, new: torch.Tensor, pos: int, block: int, fmt: str) -> None:
    """One head: rows ``new`` [t, d] to [pos, pos + t) of codes [cap, d] (float64)
    and scale [blocks] (int64), in place."""
    t, at = new.shape[0], pos
    new = new.double()
    while at < pos + t:
        blk = at // block
        lo, hi = blk * block, min((blk + 1) * block, pos + t)
        x = new[at - pos:hi - pos]
        fin = torch.isfinite(x)
        u = need(torch.where(fin, x, 0.0).abs().max().item(), fmt)
        if fmt == "int8" and not bool(fin.all()):
            u = 255
        if at > lo:
            u = max(u, int(scale[blk]))
            codes[lo:at] = round_code(codes[lo:at] * 2.0 ** (int(scale[blk]) - u), fmt)
        x = torch.where(fin, x, math.nan) * 2.0 ** (127 - u)
        codes[at:hi] = torch.nan_to_num(round_code(x, fmt)) * 0 if u == 255 else round_code(x, fmt)
        scale[blk] = u
        at = hi


def values(codes: torch.Tensor, scale: torch.Tensor, block: int) -> torch.Tensor:
    """[..., n, d] codes and [..., blocks] bytes -> values."""
    n = codes.shape[-2]
    s = torch.where(scale == 255, math.nan, torch.exp2(scale.double() - 127))
    return codes.double() * s.repeat_interleave(block, dim=-1)[..., :n, None]


def key_set(n: int, window: int, sink: int, sparse: bool) -> torch.Tensor:
    at = torch.arange(n)
    if not sparse or n <= sink + window:
        return at
    return torch.cat((at[:sink], at[n - window:]))


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n: int, scaling: float, window: int, sink: int,
           sparse: bool, sum_step: float = 0.0, query_step: float = 0.0):
    """One sequence: q [H, d], k and v [Hkv, cap, d] values.  Returns (out, spread,
    slack) [H, d]: the attention, the same weights over |v|, and what scores that are
    off by ``sum_step`` of |q| . |k| plus ``query_step`` of max|q| sum|k| (times the
    scaling) can move the attention by, to first order."""
    H, d = q.shape
    G = H // k.shape[0]
    keys = key_set(n, window, sink, sparse)
    out, spread, slack = (torch.zeros(H, d, dtype=torch.float64) for _ in range(3))
    if len(keys) == 0:
        return out, spread, slack
    for h in range(H):
        kk, vv, qq = k[h // G, keys].double(), v[h // G, keys].double(), q[h].double()
        w = torch.softmax(kk @ qq * scaling, dim=0)
        out[h] = w @ vv
        spread[h] = w @ vv.abs()
        off = (sum_step * (kk.abs() @ qq.abs()) + query_step * qq.abs().max() * kk.abs().sum(dim=1)) * scaling
        slack[h] = (w * off) @ vv.abs() + (w @ off) * spread[h]
    return out, spread, slack
