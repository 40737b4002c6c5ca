"""The decoder and the plug-in over an 8-bit KV cache, on the GPU.

The tolerances between two runs of the decoder are those of the 16-bit paths
(``test_model_gpu.py``): the two sides attend the same values, and differ by the
attention's rounding to bf16 only.
"""

import pytest
import torch

from oracle import delta_oracle as orc

pytestmark = pytest.mark.gpu

SEQ, GAMMA, WINDOW, SINK = 1024, 64, 256, 64


def _decoder(fmt, mode="dense", d=64, n_heads=8, cls=None, **kw):
    from delta_attention_b200.config import Config
    from delta_attention_b200.model import LLAMA31_8B, DeltaDecoder, tiny
    arch = tiny(LLAMA31_8B, n_layers=2, hidden=512, n_heads=n_heads, n_kv_heads=2, head_dim=d, intermediate=1024,
                vocab=1000)
    cfg = Config(delta_lambda=GAMMA, sliding_window=WINDOW, sink=SINK, mode="delta", decode_mode=mode, gamma_dec=3,
                 kv_cache=fmt, kv_block=32, **kw)
    return (cls or DeltaDecoder)(arch, cfg, device="cuda", seed=3)


def _ids(batch, n=SEQ):
    return torch.randint(0, 1000, (batch, n), generator=torch.Generator().manual_seed(5)).cuda()


def _near(a, b, what):
    err = (a.float() - b.float()).abs().max().item()
    cos = torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(), dim=0).item()
    assert err <= 5e-2 and cos >= 0.9999, f"{what}: max abs {err:.3e}, cos {cos:.6f}"


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("mode", ["dense", "sparse", "delta"])
def test_graph_decode_matches_eager_decode(mode, fmt):
    from delta_attention_b200 import ops
    from delta_attention_b200.model import DecodeGraph
    eager, graphed = _decoder(fmt, mode), _decoder(fmt, mode)
    ids, steps = _ids(2, SEQ + 13), 7
    for m in (eager, graphed):
        m.allocate_cache(2, SEQ + 13 + steps + 8)
    t0 = eager.prefill(ids)
    assert torch.equal(t0, graphed.prefill(ids))
    g = DecodeGraph(graphed, batch=2)
    g.start(t0)
    tok = t0
    for i in range(steps):
        g.step()
        h_graph = g.hidden.clone()
        h_eager = eager.forward(tok[:, None])[:, -1]
        tok = g.tok.clone()
        _near(h_graph, h_eager, f"{mode} {fmt} step {i}")
    assert graphed.length == eager.length
    g.release()
    ops.check_errors()


@pytest.mark.parametrize("fmt,d,n_heads", [("e4m3", 128, 8), ("int8", 64, 16)])
def test_decoder_attends_what_the_cache_holds(fmt, d, n_heads):
    """Prompt, single tokens, a chunk of tokens, single tokens: each step equals
    a decoder whose attention is the 64-bit oracle over the read-back cache;
    the prompt itself equals the 16-bit decoder's, bit for bit."""
    from delta_attention_b200 import ops
    from delta_attention_b200.model import DeltaDecoder

    class Reference(DeltaDecoder):
        def _attend(self, i, layer, q, k, v, prefill, n_keys=None):
            if prefill:
                return super()._attend(i, layer, q, k, v, prefill)
            kr, vr = (x.float().cpu() for x in ops.cache_read(k, n_keys=n_keys))
            s = q.shape[2]
            rows = [orc.dense_decode(q[:, :, r:r + 1].float().cpu(), kr[:, :, :n_keys - s + 1 + r],
                                     vr[:, :, :n_keys - s + 1 + r], self.scaling) for r in range(s)]
            return torch.cat(rows, dim=1).to(q.dtype).to(q.device)

    ours, ref = (_decoder(fmt, d=d, n_heads=n_heads, cls=c) for c in (DeltaDecoder, Reference))
    plain = _decoder("bf16", d=d, n_heads=n_heads)
    ids = _ids(2, SEQ + 40)
    for m in (ours, ref, plain):
        m.allocate_cache(2, SEQ + 64)
    h = ours.forward(ids[:, :SEQ])
    assert torch.equal(h, ref.forward(ids[:, :SEQ])) and torch.equal(h, plain.forward(ids[:, :SEQ]))
    at = SEQ
    for n in (1, 1, 5, 1, 31, 1):
        _near(ours.forward(ids[:, at:at + n]), ref.forward(ids[:, at:at + n]), f"{fmt} tokens [{at}, {at + n})")
        at += n
    # a new prompt into the same cache starts it afresh
    ours.prefill(ids[:, :SEQ])
    fresh = _decoder(fmt, d=d, n_heads=n_heads)
    fresh.allocate_cache(2, SEQ + 64)
    fresh.prefill(ids[:, :SEQ])
    assert ours.length == SEQ
    for x, y in zip(ours.kv8, fresh.kv8):
        assert torch.equal(x.k[:, :, :SEQ].view(torch.uint8), y.k[:, :, :SEQ].view(torch.uint8))
        assert torch.equal(x.v_scale[:, :, :SEQ // 32].view(torch.uint8), y.v_scale[:, :, :SEQ // 32].view(torch.uint8))
    ops.check_errors()


@pytest.mark.parametrize("policy", ["fixed", "drift", "drift_rel"])
def test_plugin_decode_policies_over_the_cache(policy):
    """delta_decode_forward over an 8-bit cache goes through the same schedule
    and outputs as over the 16-bit tensors that the cache reads back as."""
    from types import SimpleNamespace

    from delta_attention_b200 import ops
    from delta_attention_b200.attention import DeltaAttention
    from delta_attention_b200.kv_cache import QuantizedKV
    cfg = SimpleNamespace(num_attention_heads=8, num_key_value_heads=2, head_dim=64, sliding_window=64, sink=16,
                          decode_mode="delta", gamma_dec=4, gamma_dec_max=6, refresh_policy=policy,
                          drift_threshold=0.5, drift_k=1.0, log_drift=policy == "fixed")
    a, b = DeltaAttention(cfg), DeltaAttention(cfg)
    g = torch.Generator().manual_seed(0)
    cache = QuantizedKV.allocate(1, 2, 320, 64, format="int8", block=16)

    def draw(*shape):
        return torch.randn(*shape, generator=g).bfloat16().cuda()

    ops.cache_write(cache, draw(1, 2, 300, 64), draw(1, 2, 300, 64), pos=0)
    for i in range(16):
        n = 301 + i
        ops.cache_write(cache, draw(1, 2, 1, 64), draw(1, 2, 1, 64), pos=n - 1)
        q = draw(1, 8, 1, 64)
        k, v = ops.cache_read(cache, n_keys=n)
        got, _ = a.sdpa_rectangle_forward(a, q, cache, None, scaling=0.125, n_keys=n)
        want, _ = b.sdpa_rectangle_forward(b, q, k, v, scaling=0.125)
        assert a._dec_state["steps"] == b._dec_state["steps"], i
        # two bf16 roundings apiece (the sum with the delta) and bf16 weights on the 16-bit side
        assert (got.float() - want.float()).abs().max().item() <= 3e-2, i
    assert policy != "fixed" or len(a._dec_drift_points) == 16


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_override_over_the_cache(fmt):
    """An override gets the live keys and values as tensors, whatever the cache holds them as."""
    from delta_attention_b200 import ops
    m, plain = _decoder(fmt), _decoder(fmt)
    seen = []

    def attention(i, q, k, v, scaling, prefill):
        seen.append((i, tuple(k.shape), k.dtype, prefill))
        n, s = k.shape[2], q.shape[2]
        rows = [orc.dense_decode(q[:, :, r:r + 1].float().cpu(), k[:, :, :n - s + 1 + r].float().cpu(),
                                 v[:, :, :n - s + 1 + r].float().cpu(), scaling) for r in range(s)]
        return torch.cat(rows, dim=1).to(q.dtype).to(q.device)

    ids = _ids(2, SEQ + 9)
    for x in (m, plain):
        x.allocate_cache(2, SEQ + 32)
        x.forward(ids[:, :SEQ])
    m.attention = attention
    at = SEQ
    for n in (1, 7, 1):
        _near(m.forward(ids[:, at:at + n]), plain.forward(ids[:, at:at + n]), f"{fmt} tokens [{at}, {at + n})")
        at += n
        assert seen[-2:] == [(i, (2, 2, at, 64), torch.bfloat16, False) for i in range(2)]
    ops.check_errors()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_decode_graph_refuses_a_full_cache(fmt):
    from delta_attention_b200 import ops
    from delta_attention_b200.model import DecodeGraph
    m = _decoder(fmt)
    m.allocate_cache(1, 130)
    tok = m.prefill(_ids(1, 128))
    g = DecodeGraph(m, batch=1)
    g.start(tok)
    for _ in range(2):
        g.step()
    with pytest.raises(ValueError, match="full"):
        g.step()
    with pytest.raises(ValueError, match="full"):
        g.start(tok)
    assert m.length == 130
    g.release()
    ops.check_errors()


def test_unknown_cache_format_is_refused():
    with pytest.raises(ValueError, match="kv_cache"):
        _decoder("fp4")
