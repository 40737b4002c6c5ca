"""The 8-bit cache's calls where torch lacks the private functions that they take for speed."""

import subprocess
import sys

import pytest

WITHOUT = """
import torch
from types import SimpleNamespace
{lack}
from delta_attention_b200 import ops
from delta_attention_b200.kv_cache import QuantizedKV
"""
LACK = "del torch._C._cuda_getCurrentRawStream"


def _run(code, lack=LACK):
    run = subprocess.run([sys.executable, "-c", WITHOUT.format(lack=lack) + code], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    return run.stdout


def test_stream_without_private_functions():
    assert _run("""
torch.cuda.current_stream = lambda index: SimpleNamespace(cuda_stream=100 + index)
print(ops._raw_stream(3))
""").split() == ["103"]
    assert _run("print(ops._current_device is torch.cuda.current_device)",
                "del torch._C._cuda_getDevice").split() == ["True"]


@pytest.mark.gpu
def test_calls_without_private_functions():
    """The same values on a side stream with and without them."""
    code = """
g = torch.Generator(device="cuda").manual_seed(0)
k, v = (torch.randn(1, 2, 100, 64, generator=g, device="cuda") for _ in range(2))
q = torch.randn(1, 4, 1, 64, generator=g, device="cuda").bfloat16()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    assert ops._raw_stream(k.device.index) == side.cuda_stream and ops._current_device() == 0
    cache = QuantizedKV.allocate(1, 2, 100, 64, block=16)
    ops.cache_write(cache, k, v, pos=0)
    out = [*ops.cache_read(cache), *ops.cache_decode(q, cache, window=30, sink=2)]
side.synchronize()
for x in out:
    assert x.abs().sum() > 0
print([x.double().mul(torch.arange(x.numel(), device="cuda").view(x.shape)).sum().item() for x in out])
"""
    assert _run(code) == _run(code, "")
