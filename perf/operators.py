"""What the 8-bit key/value cache's operators are measured on.

The cache of one layer holds its keys and values as 8-bit codes (``float8_e4m3fn`` or ``int8``)
``[batch, kv_heads, capacity, dim]`` with one power-of-two scale (``float8_e8m0fnu``) for each block of
``block`` tokens and head.  The operators: writing tokens into it (``cache_write``), reading a range back
(``cache_read``) and single-token attention over it (``cache_decode``: every key, and the sink keys plus
a window).

The scale of a block is the smallest power of two ``2**e`` with ``amax / 2**e <= qmax`` (qmax 448 for
e4m3, 127 for int8), e at least -126; a write that begins inside a block never lowers that block's scale,
and where it raises it, the block's earlier codes are rounded to the new one.
"""

import math

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, op, **kw):
    c = {"op": op, "format": "e4m3", "block": 64, "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "capacity": 0, "keys": 0, "tokens": 0, "ragged": False, "dense": False, "sparse": False,
         "window": 2048, "sink": 128, "dtype": "bf16"}
    c.update(kw)
    if not c["capacity"]:
        c["capacity"] = -(-c["keys"] // c["block"]) * c["block"]
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one new token of one sequence: the write of every decode step, latency alone
        _case("write one token", "write", keys=4999, tokens=1, capacity=8192),
        # a long prompt's keys and values, written after its prefill: the bandwidth of quantising
        _case("write a prompt of 131072", "write", keys=131072, tokens=131072),
        # a padded batch of prompts with lengths of their own, appended to what each has, at a head size of 64
        _case("write a padded batch", "write", batch=6, heads=16, kv_heads=4, dim=64, keys=6021, tokens=4097,
              ragged=True, block=32, dtype="fp16"),
        # a chunk appended to a conversation, then the whole prefix read back for attention of many rows
        _case("append 513 and read back", "extend", format="int8", block=32, keys=30524, tokens=513),
        # a long prefix read back (a cache handed over to a program that wants 16 bits)
        _case("read 65536 back", "read", format="int8", keys=65536),
        # the same for a short odd prefix of a small model
        _case("read 777 back", "read", heads=8, kv_heads=2, dim=64, keys=777, block=16),
        # dense decode of one long sequence: bandwidth over the whole cache
        _case("dense decode, 131072 keys", "decode", keys=131072, dense=True),
        # the anchor step of delta decode for a batch of long prompts: both rows
        _case("anchor step, 4 x 65536", "decode", batch=4, keys=65536, dense=True, sparse=True, format="int8"),
        # the sparse step between anchors: sink and window of a long cache, latency
        _case("sparse decode, 131072 keys", "decode", keys=131072, sparse=True),
        # a short cache of a small model with odd sizes
        _case("dense decode, 777 keys", "decode", heads=8, kv_heads=1, dim=64, keys=777, block=16, dense=True),
        # a serving batch whose sequences have lengths of their own, from the longest down to none
        _case("ragged dense decode, 16", "decode", batch=16, keys=8191, capacity=16384, ragged=True, dense=True),
        # one layer's share of a decode step: the new token is written, then attended with the rest
        _case("write and attend, 32768", "step", heads=64, keys=32761, tokens=1, dense=True, sparse=True, window=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("write", "write", "extend", "read", "decode", "decode", "decode", "step"))
    dim = rng.choice((64, 128, 128))
    block = rng.choice((16, 32, 64, 64, 128))
    kv = rng.choice((1, 2, 4, 8, 8))
    heads = kv * rng.choice((1, 2, 4, 4, 8))
    batch = rng.choice((1, 1, 1, 2, 3, 4, 8))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32")) if op in ("write", "extend") else "bf16"
    most = 131072 * 8 // (kv * batch) // (2 if op == "extend" or dtype == "fp32" else 1)
    keys = _log(rng, 1, min(131072, most))
    ragged = batch > 1 and op in ("write", "decode") and rng.random() < 0.6
    tokens = 0
    if op in ("write", "extend"):
        tokens = 1 if rng.random() < 0.3 else _log(rng, 1, keys)
    elif op == "step":
        tokens = 1
    dense = op in ("decode", "step") and rng.random() < 0.7
    sparse = op in ("decode", "step") and (not dense or rng.random() < 0.5)
    room = rng.choice((0, 0, 1, 7))
    return _case(None, op, format=rng.choice(("e4m3", "e4m3", "int8")), block=block, batch=batch, heads=heads,
                 kv_heads=kv, dim=dim, keys=keys, tokens=tokens, ragged=ragged, dense=dense, sparse=sparse,
                 capacity=(-(-keys // block) + room) * block, window=rng.choice((64, 500, 2048, 4096)),
                 sink=rng.choice((0, 4, 128, 1024)), dtype=dtype)


def _spread(most, batch):
    """Lengths from ``most`` down to 0 where a batch has lengths of its own."""
    return [most * (batch - 1 - i) // (batch - 1) for i in range(batch)]


def _lengths(case):
    """(keys of each sequence once the call is done, new tokens of each)."""
    b, n, t = case["batch"], case["keys"], case["tokens"]
    if not case["ragged"]:
        return [n] * b, [t] * b
    if case["op"] == "decode":
        return _spread(n, b), [0] * b
    new = _spread(t, b)
    return [n - t + x for x in new], new


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    b, H, Hkv, d, cap, block = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "capacity", "block"))
    keys, new = _lengths(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    def key_like(n):  # keys have a few strong channels and a magnitude that varies from token to token
        return normal(b, Hkv, n, d) * torch.exp(0.5 * normal(1, Hkv, 1, d)) * torch.exp(0.3 * normal(b, 1, n, 1))

    def value_like(n):
        return 0.5 * normal(b, Hkv, n, d) * torch.exp(0.3 * normal(b, 1, n, 1))

    s = {"case": case}
    s["k"], s["k_scale"] = _quantise(key_like(cap), block, case["format"])
    s["v"], s["v_scale"] = _quantise(value_like(cap), block, case["format"])
    if case["tokens"]:
        dt = FLOATS[case["dtype"]]
        # token-major in memory, as a projection's output is, and seen head by head
        s["k_new"] = key_like(case["tokens"]).transpose(1, 2).to(dt).contiguous().transpose(1, 2)
        s["v_new"] = value_like(case["tokens"]).transpose(1, 2).to(dt).contiguous().transpose(1, 2)
        s["pos"] = keys[0] - new[0]
        s["new"] = torch.tensor(new, dtype=torch.int32, device=dev) if case["ragged"] else None
    if case["dense"] or case["sparse"]:
        s["q"] = (1.5 * normal(b, H, 1, d)).to(torch.bfloat16)
        s["lengths"] = torch.tensor(keys, dtype=torch.int32, device=dev) if case["ragged"] else None
    if own:
        from delta_attention_b200.kv_cache import QuantizedKV

        s["cache"] = QuantizedKV(s["k"], s["v"], s["k_scale"], s["v_scale"], block)
    return s


# ---- the plain form -----------------------------------------------------------------------------

def _need(amax, fmt):
    """Biased exponent of the smallest power of two s with amax / s <= qmax (int32, at least 1)."""
    m, e = torch.frexp(amax / QMAX[fmt])  # amax / qmax = m * 2**e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, e + 127, torch.ones_like(e)).clamp_min(1)


def _to_codes(x, fmt):
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(x).clamp(-127, 127).to(torch.int8)


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _quantise(x, block, fmt):
    b, h, n, d = x.shape
    x = x.reshape(b, h, n // block, block, d)
    u = _need(x.abs().amax(dim=(3, 4)), fmt)
    codes = _to_codes(x * _pow2(127 - u)[..., None, None], fmt)
    return codes.reshape(b, h, n, d), u.to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_write(new, codes, scale, pos, lengths, block, fmt):
    """The new rows [b, h, t, d] go to [pos, pos + lengths) of codes and scale, in place."""
    b, h, t, d = new.shape
    cap = codes.shape[2]
    blocks = min((t + 2 * block - 2) // block, cap // block)
    first = min(pos // block, cap // block - blocks)
    at = torch.arange(first * block, (first + blocks) * block, device=new.device)
    end = pos + (torch.full((b,), t, device=new.device) if lengths is None else lengths)
    fresh = ((at >= pos) & (at < end[:, None]))[:, None, :, None]
    x = torch.where(fresh, new[:, :, (at - pos).clamp(0, t - 1)].float(), 0.0)
    shape = (b, h, blocks, block, d)
    u_old = scale.view(torch.uint8)[:, :, first:first + blocks].int()
    starts = torch.arange(first, first + blocks, device=new.device) * block
    held = starts < pos                      # blocks with tokens before pos
    u = _need(x.abs().reshape(shape).amax(dim=(3, 4)), fmt)
    u = torch.where(held, torch.maximum(u, u_old), u)
    touched = (starts + block > pos) & (starts < end[:, None])
    u = torch.where(touched[:, None], u, u_old)
    old = codes[:, :, first * block:(first + blocks) * block]
    kept = old.float().reshape(shape) * _pow2(u_old - u)[..., None, None]
    fresh_codes = _to_codes(x.reshape(shape) * _pow2(127 - u)[..., None, None], fmt).reshape(old.shape)
    kept_codes = _to_codes(kept, fmt).reshape(old.shape)
    before = (at < pos)[:, None]
    out = torch.where(fresh, fresh_codes.view(torch.uint8),
                      torch.where(before, kept_codes.view(torch.uint8), old.view(torch.uint8)))
    old.view(torch.uint8).copy_(out)
    scale.view(torch.uint8)[:, :, first:first + blocks] = u.to(torch.uint8)


def _plain_values(codes, scale, block, at):
    """The values at the positions ``at`` ([n], or [b, 1, n] where each sequence has its own), fp32."""
    u = scale.view(torch.uint8)
    if at.dim() == 1:
        c, e = codes.view(torch.uint8)[:, :, at], u[:, :, at // block]
    else:
        b, h = codes.shape[:2]
        i, j = torch.arange(b, device=at.device)[:, None, None], torch.arange(h, device=at.device)[:, None]
        c, e = codes.view(torch.uint8)[i, j, at], u[i, j, at // block]
    return c.view(codes.dtype).float() * _pow2(e.int() - 127)[..., None]


def _plain_attend(q, k, v, live):
    """q [b, h, g, d] over k and v [b, h, n, d], of which the first ``live`` [b, 1] rows count."""
    x = (q @ k.transpose(2, 3)) * q.shape[-1] ** -0.5
    x = x.masked_fill(~(torch.arange(k.shape[2], device=q.device) < live)[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    o = (p @ v) / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    return o.flatten(1, 2)[:, None].to(torch.bfloat16)


def _plain_decode(s, n):
    c, block = s["case"], s["case"]["block"]
    b, H, _, d = s["q"].shape
    q = s["q"].float().reshape(b, c["kv_heads"], -1, d)
    live = torch.full((b, 1), n, device=q.device) if s["lengths"] is None else s["lengths"][:, None]
    out = {}
    if c["dense"]:
        at = torch.arange(n, device=q.device)
        out["dense"] = _plain_attend(q, *(_plain_values(s[x], s[x + "_scale"], block, at) for x in ("k", "v")), live)
    if c["sparse"]:
        near = c["sink"] + c["window"]
        t = torch.arange(min(n, near), device=q.device)
        at = torch.where((live > near) & (t >= c["sink"]), live - near + t, t)[:, None]
        out["sparse"] = _plain_attend(q, *(_plain_values(s[x], s[x + "_scale"], block, at) for x in ("k", "v")),
                                      live.clamp_max(near))
    return out


def run(state):
    s, c = state, state["case"]
    op, n = c["op"], c["keys"]
    if own:
        from delta_attention_b200 import ops
    if op in ("write", "extend", "step"):
        if own:
            ops.cache_write(s["cache"], s["k_new"], s["v_new"], pos=s["pos"], lengths=s["new"])
        else:
            _plain_write(s["k_new"], s["k"], s["k_scale"], s["pos"], s["new"], c["block"], c["format"])
            _plain_write(s["v_new"], s["v"], s["v_scale"], s["pos"], s["new"], c["block"], c["format"])
    out = {}
    if op in ("extend", "read"):
        if own:
            out["k"], out["v"] = ops.cache_read(s["cache"], n_keys=n)
        else:
            at = torch.arange(n, device=s["k"].device)
            out["k"], out["v"] = (_plain_values(s[x], s[x + "_scale"], c["block"], at).to(torch.bfloat16)
                                  for x in ("k", "v"))
    if op in ("decode", "step"):
        if own:
            dense, sparse = ops.cache_decode(s["q"], s["cache"], window=c["window"], sink=c["sink"],
                                             want_dense=c["dense"], want_sparse=c["sparse"], n_keys=n,
                                             n_keys_dev=s["lengths"])
            out.update({x: o for x, o in (("dense", dense), ("sparse", sparse)) if o is not None})
        else:
            out.update(_plain_decode(s, n))
    if op in ("write", "step"):
        out.update({x: s[x] for x in ("k", "v", "k_scale", "v_scale")})
    return out


def work(case):
    keys, new = _lengths(case)
    H, Hkv, d, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    op, size = case["op"], {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    bytes_, flops = 0, 0
    for n, t in zip(keys, new):
        if t:  # each new value read once and its code written once, and the scales of the touched blocks
            bytes_ += 2 * Hkv * (t * d * (size + 1) + (n - 1) // block - (n - t) // block + 1)
            flops += 2 * Hkv * t * d * 2
        if op in ("extend", "read"):
            bytes_ += 2 * Hkv * (n * d * 3 + -(-n // block))
            flops += 2 * Hkv * n * d
        if op in ("decode", "step"):
            seen = n if case["dense"] else min(n, case["sink"] + case["window"])
            bytes_ += 2 * Hkv * (seen * d + -(-seen // block)) + H * d * 2 * (1 + case["dense"] + case["sparse"])
            rows = n * case["dense"] + min(n, case["sink"] + case["window"]) * case["sparse"]
            flops += 4 * H * d * rows
    return {"bytes": bytes_, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_round(x, fmt):
    """The nearest value that the format has, ties to the even code; x within the format's range."""
    if fmt == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_scale(amax, fmt):
    s = torch.exp2(torch.ceil(torch.log2(amax.clamp_min(2.0 ** -140) / QMAX[fmt])).clamp_min(-126.0))
    s = torch.where(amax / s > QMAX[fmt], 2 * s, s)
    return torch.where((amax / (s / 2) <= QMAX[fmt]) & (s > 2.0 ** -126), s / 2, s)


def _exact_write(codes, scale, new, pos, count, block, fmt):
    """codes [h, n, d] and scale [h, blocks] of one sequence, float64, after the write."""
    at = pos
    while at < pos + count:
        blk = at // block
        lo, hi = blk * block, min((blk + 1) * block, pos + count)
        x = new[:, at - pos:hi - pos]
        s = _exact_scale(x.abs().amax(dim=(1, 2)), fmt)
        if at > lo:
            s = torch.maximum(s, scale[:, blk])
            codes[:, lo:at] = _exact_round(codes[:, lo:at] * (scale[:, blk] / s)[:, None, None], fmt)
        codes[:, at:hi] = _exact_round(x / s[:, None, None], fmt)
        scale[:, blk] = s
        at = hi


def exact(case, seed):
    if case["tokens"] > 16384:
        # a long write has one step of this loop for each block: the whole blocks at once instead
        whole = case["keys"] == case["tokens"] and not case["ragged"]
        if not whole:
            return None
    s = prepare(case, seed)
    block, fmt, n, d = case["block"], case["format"], case["keys"], case["dim"]
    keys, new = _lengths(case)
    code, scale = {}, {}
    for x in ("k", "v"):
        code[x] = s[x].double()
        scale[x] = torch.exp2(s[x + "_scale"].view(torch.uint8).double() - 127)
        for i in range(case["batch"]):
            if new[i] > 16384:
                c = new[i] // block * block
                y = s[x + "_new"][i, :, :c].double().reshape(case["kv_heads"], c // block, block, d)
                z = _exact_scale(y.abs().amax(dim=(2, 3)), fmt)
                code[x][i, :, :c] = _exact_round(y / z[..., None, None], fmt).flatten(1, 2)
                scale[x][i, :, :c // block] = z
                _exact_write(code[x][i], scale[x][i], s[x + "_new"][i, :, c:].double(), c, new[i] - c, block, fmt)
            elif new[i]:
                _exact_write(code[x][i], scale[x][i], s[x + "_new"][i].double(), s["pos"], new[i], block, fmt)
    out = {}
    op = case["op"]
    if op in ("write", "step"):
        for x in ("k", "v"):
            out[x], out[x + "_scale"] = code[x], scale[x]
    if op == "write":
        return out
    place = torch.arange(case["capacity"], device=s["k"].device) // block
    value = {x: code[x] * scale[x][:, :, place][..., None] for x in ("k", "v")}
    if op in ("extend", "read"):
        return {x: value[x][:, :, :n] for x in ("k", "v")}
    group = case["heads"] // case["kv_heads"]
    for name in ("dense", "sparse"):
        if not case[name]:
            continue
        rows = torch.zeros(case["batch"], 1, case["heads"], d, dtype=torch.float64, device=s["q"].device)
        for i in range(case["batch"]):
            live = keys[i]
            seen = torch.arange(live, device=s["q"].device)
            if name == "sparse" and live > case["sink"] + case["window"]:
                seen = torch.cat((seen[:case["sink"]], seen[live - case["window"]:]))
            if len(seen) == 0:
                continue
            for h in range(case["kv_heads"]):
                q = s["q"][i, h * group:(h + 1) * group, 0].double()
                w = torch.softmax(q @ value["k"][i, h, seen].T / math.sqrt(d), dim=-1)
                rows[i, 0, h * group:(h + 1) * group] = w @ value["v"][i, h, seen]
        out[name] = rows
    return out
