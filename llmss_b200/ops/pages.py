"""Cache pages in 8 bits: codes and a 32-bit scale per token and head.

A page holds what the 16-bit pages hold, [num_blocks, kv_heads, block_size, head_dim], in a byte per value; ``scale`` [num_blocks, kv_heads,
block_size] turns a row's codes into numbers, value = code * scale (scales are 0 or more, or NaN).  One scale per row, because a row is written once, by
one warp, when its token comes, and nothing that is in the cache has to be read or changed for it.  Integers (``torch.int8``) have even steps of 1 / 127 of
a row's largest value, which suits rows whose values are of one size; ``torch.float8_e4m3fn`` has steps of 1 / 16 of each value, which suits rows with a
few large ones.
"""
from __future__ import annotations

import torch

FORMATS = {torch.int8: 1, torch.float8_e4m3fn: 2}           # ids of the kernel library
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
NAMES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


class QuantPages:
    """Keys or values of one layer; passes for the page tensor in ``ops.rope_kv_write`` and ``ops.attention``."""

    __slots__ = ("data", "scale")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor):
        if data.dtype not in FORMATS:
            raise TypeError(f"QuantPages: pages are int8 or float8_e4m3fn, got {data.dtype}")
        if scale.dtype is not torch.float32 or data.dim() != 4 or scale.shape != data.shape[:3]:
            raise ValueError(f"QuantPages: pages [blocks, heads, block, d] with 32-bit scales [blocks, heads, block], got {tuple(data.shape)} and "
                             f"{scale.dtype} {tuple(scale.shape)}")
        if not (data.is_contiguous() and scale.is_contiguous()):
            raise ValueError("QuantPages: pages and scales must be contiguous")
        if data.get_device() != scale.get_device():
            raise ValueError(f"QuantPages: pages on {data.device}, scales on {scale.device}")
        self.data, self.scale = data, scale

    @property
    def shape(self):
        return self.data.shape

    @property
    def dtype(self):
        return self.data.dtype

    def values(self, dtype=torch.float32) -> torch.Tensor:
        """The numbers that the codes stand for."""
        return (self.data.float() * self.scale[..., None]).to(dtype)


def quantise(x: torch.Tensor, dtype):
    """Codes and scales of rows [..., d]: scale = max |x| / largest code (32-bit division), code = x / scale rounded to the nearest (ties to even).
    A row of zeros has scale 0; one that holds a NaN or an infinity has scale NaN and reads back as NaN."""
    x = x.float()
    amax = x.abs().amax(-1)
    # a tensor below the line: torch divides by a plain number on the GPU through its reciprocal, which rounds twice
    scale = torch.where(torch.isfinite(x).all(-1), amax / torch.full_like(amax, QMAX[dtype]), torch.nan)
    y = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0).clamp(-QMAX[dtype], QMAX[dtype]) + 0.0      # -0 becomes 0
    return (y.round().to(dtype) if dtype == torch.int8 else y.to(dtype)), scale
