"""Serving from packed block formats (new; the reference has none): products with 4-bit weights, a paged cache of K and V in
MX format, and attention over it.

These are the operators that read the codes which ``mx_quantize`` and ``nvfp4_quantize`` hand out.  Dense tensors are float32,
bfloat16 or float16; sums, softmax statistics and scales are held in 32 bits and a result is rounded to its type once.  The
operands of the products have 16 bits: rows of x and q in bfloat16 and float16 are held exactly down to 2^-29 of their largest
magnitude and to 2^-39 of it below, float32 ones to 22 bits and 2^-50; the weights of a softmax to 11 bits (chunks of 32 rows and
more: 8 in bfloat16, 16 in float16, 24 in float32; fewer rows in float32: 22), and at least to 2^-26 of the row's largest.  They
answer with a model and do not train it: an input that needs a gradient is refused while gradients are recorded, and so is one
that carries a forward-mode tangent.

The tokens of a batch.  ``pages`` [sequences, width] names for each sequence the pages that hold its tokens, in order (an entry
outside the cache holds none: -1 behind the last page); ``lens`` [sequences] counts a sequence's tokens with the new ones.  New
rows come either as [sequences, new, heads, head_dim], or, for a ragged batch, as [rows, heads, head_dim] with ``starts``
[sequences + 1]: sequence s has the rows starts[s] to starts[s + 1].  Row i of a sequence's n stands at position
``lens[s] - n + i``; where that is negative (a padded sequence) it stands nowhere: it is not written, and reads and attends to
nothing.  All three are int32.
"""
from __future__ import annotations

import math
from typing import Literal, NamedTuple

import torch

from .. import backend as _be

__all__ = ["mx_linear", "nvfp4_linear", "MXCache", "mx_cache_write", "mx_cache_read", "mx_attention"]


def mx_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T + bias`` with W [out, in] in MXFP4, as ``mx_quantize(w, "e2m1", 32, return_scales=True, return_codes=True)``
    packs it: ``codes`` [out, in / 2], ``scales`` [out, in / 32].  ``in`` is a multiple of 32; x has any number of rows."""
    return _be.mx_linear(x, codes, scales, bias)


def nvfp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, global_scale: torch.Tensor | float,
                 bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T + bias`` with W [out, in] in NVFP4, as ``nvfp4_quantize(w, return_scales=True, return_codes=True)`` packs it:
    ``codes`` [out, in / 2], ``scales`` the E4M3 bytes [out, in / 16], ``global_scale`` the tensor scale (one float32 value on
    the GPU, or a number).  ``in`` is a multiple of 32; x has any number of rows."""
    if not isinstance(global_scale, torch.Tensor):
        global_scale = torch.full((1,), float(global_scale), dtype=torch.float32, device=x.device)
    return _be.nvfp4_linear(x, codes, scales, global_scale, bias)


class MXCache(NamedTuple):
    """K and V of one layer in pages, quantized along head_dim in blocks of 32 (MXFP8 or MXFP4): codes and E8M0 scale bytes of
    each.  The functions below also take a plain tuple of the four tensors.  Codes that are NaN stand in blocks whose scale byte is
    0xFF, and codes times their scales do not pass float32's range, as ``mx_cache_write`` leaves them."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, elem_format: Literal["e4m3", "e2m1"] = "e4m3", device="cuda"):
        """A cache of zeros with ``pages`` pages of ``page`` tokens each (a power of two from 8 to 256); head_dim is a multiple
        of 32 up to 256."""
        if elem_format not in ("e4m3", "e2m1"):
            raise ValueError("elem_format must be 'e4m3' or 'e2m1'")
        if head_dim < 32 or head_dim > 256 or head_dim % 32:
            raise ValueError("head_dim must be a multiple of 32 up to 256")
        if page < 8 or page > 256 or page & (page - 1):
            raise ValueError("page must be a power of two from 8 to 256")
        width = head_dim if elem_format == "e4m3" else head_dim // 2
        return cls(*(torch.zeros(pages, kv_heads, page, n, dtype=torch.uint8, device=device) for n in (width, head_dim // 32) * 2))


def mx_cache_write(k: torch.Tensor, v: torch.Tensor, cache, pages: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor | None = None) -> None:
    """Quantizes the new rows of K and V into the cache, in place: the codes and scales of ``mx_quantize`` on the same values.
    The last dimension of k and v is contiguous (or is made so); the others may have any strides.  Where two rows of a call
    stand in the same place of the same page, which bytes of which are kept is not defined."""
    _be.mx_cache_write(k, v, cache, pages, lens, starts)


def mx_cache_read(cache, pages: torch.Tensor, lens: torch.Tensor, rows: int, starts: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The last ``rows`` tokens of each sequence (with ``starts``: the rows that it describes, ``rows`` in all) as K and V of
    ``dtype``; zeros for a row that stands nowhere."""
    return _be.mx_cache_read(cache, pages, lens, rows, starts, dtype)


def mx_attention(q: torch.Tensor, cache, pages: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor | None = None, scale: float | None = None,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens over their sequences' tokens in the cache, the new ones included (write them first).

    q [sequences, new, heads, head_dim], or [rows, heads, head_dim] with ``starts``; query head h reads kv head
    ``h // (heads / kv_heads)``; ``scale`` is 1 / sqrt(head_dim) unless given.  With ``window`` a token sees the last ``window``
    positions, its own among them, and the first ``sinks`` ones.  A row that sees nothing gives zeros.  ``out`` takes the result
    and may be q itself or share memory with it; its rows behind the last sequence are left as they were."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.shape[-1] else 1.0
    return _be.mx_attention(q, cache, pages, lens, starts, float(scale), window, sinks, out)
