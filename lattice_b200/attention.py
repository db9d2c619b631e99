"""Objects that the attention half of a step is called with: rotary frequencies and a paged key/value cache.

The calls themselves are methods of ``CudaQ4Backend`` (``rope_rows``, ``kv_append``), beside the projections
that stand before and behind them.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import KvCacheDesc, RopeDesc, RopeScaling, check

_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}
_SCALINGS = {"plain": _lib.ROPE_PLAIN, "linear": _lib.ROPE_LINEAR, "ntk": _lib.ROPE_NTK, "yarn": _lib.ROPE_YARN,
             "bands": _lib.ROPE_BANDS}


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
                     original_len: float = 4096.0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """``(freq, scale)``: radians a position of each pair (numpy f64, ``rot_dim / 2``) and the factor of the
    rotated entries.  ``scaling``: "plain", "linear", "ntk", "yarn" or "bands" (see ``lq4_rope_frequencies``)."""
    if scaling not in _SCALINGS:
        raise ValueError(f"unknown rotary scaling {scaling!r}; one of {sorted(_SCALINGS)}")
    freq = np.zeros(max(rot_dim // 2, 1), np.float64)
    scale = C.c_float()
    desc = RopeScaling(_SCALINGS[scaling], rot_dim, theta, factor, original_len, beta_fast, beta_slow)
    check(_lib.lib().lq4_rope_frequencies(C.byref(desc), freq.ctypes.data, C.byref(scale)))
    return freq, float(scale.value)


class RopeTable:
    """Frequencies on the device (f64, one per pair), how a pair lies in a head, and the scale of rotated entries."""

    __slots__ = ("freq", "desc", "address", "device")

    def __init__(self, freq: torch.Tensor, layout: str = "half", scale: float = 1.0):
        if layout not in _LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}; one of {sorted(_LAYOUTS)}")
        if freq.dtype != torch.float64 or freq.dim() != 1 or not freq.is_contiguous() or not freq.is_cuda:
            raise TypeError("freq must be a contiguous 1-D float64 device tensor, one entry per pair")
        self.freq = freq
        self.desc = RopeDesc(freq.data_ptr(), 2 * freq.numel(), _LAYOUTS[layout], scale)
        self.address, self.device = C.addressof(self.desc), freq.get_device()

    @classmethod
    def from_config(cls, rot_dim: int, device, layout: str = "half", **scaling) -> "RopeTable":
        """Frequencies as ``rope_frequencies(rot_dim, **scaling)`` gives them, on ``device``."""
        freq, scale = rope_frequencies(rot_dim, **scaling)
        return cls(torch.from_numpy(freq).to(device), layout, scale)


class KvCache:
    """One layer's paged cache: ``k`` and ``v`` are ``[pages, page_size, kv_heads, head_dim]`` bf16 device tensors
    (any strides but the innermost, the same for both: a ``[pages, kv_heads, page_size, head_dim]`` allocation comes
    as its transposed view), ``page_table`` is ``[batch, max_pages]`` int32.  The tensors are referenced, not copied."""

    __slots__ = ("k", "v", "page_table", "desc", "address", "device", "rows_shape")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor):
        if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise TypeError(f"the cache holds bfloat16, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must be [pages, page_size, kv_heads, head_dim] with equal strides, the innermost 1")
        pages, size, heads, dim = k.shape
        s0, s1, s2, _ = k.stride()
        if (not s0 and pages > 1) or (not s1 and size > 1) or (not s2 and heads > 1):      # (0 means dense to the library)
            raise ValueError("k and v must not be expanded tensors")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or not page_table.is_contiguous():
            raise TypeError("page_table must be a contiguous [batch, max_pages] int32 tensor")
        self.device = k.get_device()
        if self.device < 0 or v.get_device() != self.device or page_table.get_device() != self.device:
            raise ValueError("k, v and page_table must lie on one CUDA device")
        self.k, self.v, self.page_table = k, v, page_table
        batch, max_pages = page_table.shape
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), pages, size, heads, dim, s0 if pages > 1 else 0, s1 if size > 1 else 0,
                                s2 if heads > 1 else 0, page_table.data_ptr(), batch, max_pages)      # (of one entry a stride may be anything)
        self.address = C.addressof(self.desc)
        self.rows_shape = (batch, heads, dim)                            # of rows to append or attend with, but for their number

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, page_table: torch.Tensor) -> "KvCache":
        """A zeroed dense cache on ``page_table``'s device."""
        shape = (pages, page_size, kv_heads, head_dim)
        return cls(torch.zeros(shape, dtype=torch.bfloat16, device=page_table.device),
                   torch.zeros(shape, dtype=torch.bfloat16, device=page_table.device), page_table)
