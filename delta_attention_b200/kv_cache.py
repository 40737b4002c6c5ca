"""The 8-bit KV cache of one layer: codes, and a power-of-two scale per block of
tokens and head.

``QuantizedKV`` holds the tensors that ``ops.cache_write``, ``ops.cache_read``
and ``ops.cache_decode`` work on.  A code ``c`` of a block whose scale is ``s``
stands for ``c * s``; the formats are ``e4m3`` (``float8_e4m3fn``, relative
rounding of at most 2^-4) and ``int8`` (rounding of at most ``s / 2``).  The
scale of a block is the smallest power of two that brings the block's largest
magnitude within the format (448 or 127).  A block keeps one scale while tokens
are appended to it: it only rises, and the codes already there are rounded to
the new scale (exactly, but for e4m3 codes that leave the normal range and for
int8 codes that lose their last bit).
"""

from __future__ import annotations

import torch

from ._lib import ABI_VERSION, CACHE_FORMATS, CacheDecodeArgs, CacheReadArgs, CacheWriteArgs

BLOCKS = (16, 32, 64, 128)
CODE_TYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SCALE_TYPE = torch.float8_e8m0fnu
_FORMATS = {t: f for f, t in CODE_TYPES.items()}


class QuantizedKV:
    """``k``, ``v`` [b, Hkv, capacity, d] (``float8_e4m3fn`` or ``int8``, d 64 or
    128 and contiguous, other strides multiples of 16 bytes) and ``k_scale``,
    ``v_scale`` [b, Hkv, ceil(capacity / block)] (``float8_e8m0fnu``).  The tensors
    are written in place by ``ops.cache_write``; they are kept as they are given
    (no copy), so they must stay where they are while the object is used."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 block: int = 64):
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"codes must be two [b, Hkv, capacity, d] tensors, got {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
        if k.dtype not in _FORMATS or v.dtype != k.dtype:
            raise ValueError(f"codes must both be float8_e4m3fn or int8, got {k.dtype} and {v.dtype}")
        b, Hkv, cap, d = k.shape
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block}")
        if d not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {d}")
        if min(b, Hkv, cap) <= 0:
            raise ValueError(f"empty cache {tuple(k.shape)}")
        want = (b, Hkv, -(-cap // block))
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if tuple(t.shape) != want or t.dtype != SCALE_TYPE:
                raise ValueError(f"{name} must be {want} {SCALE_TYPE}, got {tuple(t.shape)} {t.dtype}")
            if (t.stride(2) != 1 and want[2] > 1) or (t.stride(1) <= 0 and Hkv > 1) or (t.stride(0) <= 0 and b > 1):
                raise ValueError(f"{name} must have contiguous blocks and positive strides, got {t.stride()}")
        for name, t in (("k", k), ("v", v)):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(
                    n > 1 and (st <= 0 or st % 16) for n, st in zip(t.shape, t.stride()[:3])):
                raise ValueError(f"{name} must have d contiguous, and a base and other strides that are multiples "
                                 f"of 16 bytes, got {t.stride()}")
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1:
            raise ValueError("the cache's tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale, self.block = k, v, k_scale, v_scale, int(block)
        self.format = _FORMATS[k.dtype]
        self.batch, self.n_kv_heads, self.capacity, self.head_dim = b, Hkv, cap, d
        self.device = k.device
        self.index = k.device.index if k.device.type == "cuda" else None
        self.workspace_bytes = {}  # of cache_decode, by (heads, window, sink)
        if self.index is not None:
            from .ops import error_word

            self.error_word = error_word(self.device)  # (here, not in a call that a graph may be capturing)
        # the C ABI's argument structs with this cache filled in; each call copies one
        self._write_args, self._read_args, self._decode_args = CacheWriteArgs(), CacheReadArgs(), CacheDecodeArgs()
        for a in (self._write_args, self._read_args, self._decode_args):
            a.abi_version = ABI_VERSION
            self._describe(a.cache)

    def _describe(self, c) -> None:
        c.batch, c.n_kv_heads, c.capacity, c.head_dim = self.batch, self.n_kv_heads, self.capacity, self.head_dim
        c.block, c.format = self.block, CACHE_FORMATS[self.format]
        for name in ("k", "v"):
            t, s = getattr(self, name), getattr(self, name + "_scale")
            setattr(c, name, t.data_ptr())
            setattr(c, name + "_scale", s.data_ptr())
            for axis, n, st in zip("bhs", t.shape, t.stride()):  # a size-1 axis gets a harmless legal stride
                setattr(c, f"{name}_stride_{axis}", st if n > 1 else self.head_dim)
            for axis, n, st in zip("bh", s.shape, s.stride()):
                setattr(c, f"{name}_scale_stride_{axis}", st if n > 1 else 1)

    @classmethod
    def allocate(cls, batch: int, n_kv_heads: int, capacity: int, head_dim: int, *, format: str = "e4m3",
                 block: int = 64, device="cuda") -> "QuantizedKV":
        """An empty cache (codes and scales zero)."""
        if format not in CODE_TYPES:
            raise ValueError(f"unknown cache format {format!r} (one of {', '.join(CODE_TYPES)})")
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block}")
        shape, blocks = (batch, n_kv_heads, capacity, head_dim), -(-capacity // block)

        def zeros(size, dtype):
            return torch.zeros(size, dtype=torch.uint8, device=device).view(dtype)

        return cls(zeros(shape, CODE_TYPES[format]), zeros(shape, CODE_TYPES[format]),
                   zeros(shape[:2] + (blocks,), SCALE_TYPE), zeros(shape[:2] + (blocks,), SCALE_TYPE), block)

    def nbytes(self) -> int:
        """Bytes of the codes and scales."""
        return sum(t.numel() for t in (self.k, self.v, self.k_scale, self.v_scale))

