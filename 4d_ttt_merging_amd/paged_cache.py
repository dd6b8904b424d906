"""A cache of keys and values in 4 bits, in pages, and attention over it, on gfx950.

A scene that grows frame by frame keeps the keys and values of every layer; a step reads all of them, so their
bytes are its time.  `cache_append` stores new tokens (rotating keys, and queries beside them, on the way),
`cached_attention` attends over what is stored, `cache_read` gives tokens back as numbers
(csrc/paged_cache.hip, csrc/cached_attention.hip).  Inference only; neither a CPU path nor a counterpart in the
reference, whose attention takes the keys of one call (vggt_omega/models/mass_bias_attention.py:85-129).

The format is the OCP one of E2M1 codes with an E8M0 scale for 32 channels of a token and head (17/32 byte a
channel of a key or value): the scale is the smallest power of two, from 2**-125 to 2**125, of which 7 are at least the
largest magnitude, each channel the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times that (ties to the even code), so none is off
by more than the scale.  A block of 32 channels with one that is not finite reads as NaN.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib


class PagedCache(NamedTuple):
    """The memory of a cache: `data` uint8 [pages, kv_heads, page_size / 32, 34 * head_dim] and, for tokens with
    masses, `log_mass` fp32 [pages, page_size].  Which pages a sequence holds, and how many tokens, is the
    caller's: a page table (int32 [batch, pages of the longest]) and lengths (int32 [batch]) go with every call."""

    data: torch.Tensor
    log_mass: torch.Tensor | None = None

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, masses: bool = False,
              device: torch.device | str = "cuda") -> "PagedCache":
        """A cache of zeros.  head_dim 64 or 128; page_size a power of two, 32 to 1,024."""
        if head_dim not in (64, 128):
            raise ValueError("a paged cache takes 64 or 128 channels a head")
        if page_size < 32 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("the page size must be a power of two from 32 to 1,024")
        if pages < 0 or kv_heads < 1:
            raise ValueError("a paged cache has pages and key heads")
        data = torch.zeros((pages, kv_heads, page_size // 32, 34 * head_dim), dtype=torch.uint8, device=device)
        return cls(data, torch.zeros((pages, page_size), device=device) if masses else None)

    @property
    def page_size(self) -> int:
        return 32 * self.data.shape[2]

    @property
    def kv_heads(self) -> int:
        return self.data.shape[1]

    @property
    def head_dim(self) -> int:
        return self.data.shape[3] // 34


def _ready(*tensors: torch.Tensor | None) -> None:
    try:
        _lib.load()
    except _lib.ExtensionUnavailable as error:
        raise RuntimeError(str(error)) from error
    _lib.require_gpu(*tensors)


def _autocast(*tensors: torch.Tensor | None) -> tuple[torch.Tensor | None, ...]:
    """fp32 operands in the autocast type, where that is a 16-bit one."""
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        if dtype in (torch.bfloat16, torch.float16):
            return tuple(t.to(dtype) if t is not None and t.dtype == torch.float32 else t for t in tensors)
    return tensors


def cache_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                 counts: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
                 rope: tuple[torch.Tensor, torch.Tensor] | None = None, positions: torch.Tensor | None = None,
                 log_mass: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store new tokens of every sequence in their pages; returns q rotated (None without q).

    k, v [B, Hk, N, D] of one type (bf16, f16 or fp32), any strides; token i of sequence b goes to place
    starts[b] + i (int32 [B]); from counts[b] on (int32 [B], default N) tokens are padding and are left out.
      rope       (sin, cos), floating [rows, D]: keys are stored, and q [B, H, N, D] is returned (rounded to its type,
                 its padding as zeros, token-major in memory where q is), as x cos + (-x[D/2:], x[:D/2]) sin
      positions  int32 [B, N]: the tables' row of a token; default its place.  Tokens with no such row (a frame's
                 special tokens: -1) are not rotated
      log_mass   floating [B, N]: added to every score of the token, for caches with masses; default zeros
    A rotated key's codes are the nearest to the exact values; q is rotated in fp32.  Tokens past the page table, or
    whose entry is not a page of the cache (-1, say), are left out.  Two tokens of one call must not have
    the same place in the cache.  Under bf16 or f16 autocast fp32 operands are cast first."""
    _ready(cache.data, cache.log_mass, k, v, q, page_table, starts, counts, positions, log_mass, *(rope or ()))
    if positions is not None and rope is None:
        raise ValueError("positions go with rope")
    k, v, q = _autocast(k, v, q)
    sin, cos = rope if rope is not None else (None, None)
    out = torch.ops.vgo.cache_append(k, v, q, cache.data, cache.log_mass, page_table, starts, counts, sin, cos, positions,
                                     log_mass)
    return None if q is None else out


def cache_read(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor, n_tokens: int,
               counts: torch.Tensor | None = None, *, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens starts[b] .. starts[b] + n_tokens - 1 of every sequence as numbers: k, v [B, Hk, n_tokens, D], exact in
    bf16 and fp32.  Zeros from counts[b] on and for tokens that have no page."""
    _ready(cache.data, page_table, starts, counts)
    return torch.ops.vgo.cache_read(cache.data, page_table, starts, counts, n_tokens, dtype)


def cached_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                     counts: torch.Tensor | None = None, *, causal: bool = False, scale: float | None = None) -> torch.Tensor:
    """Attention of q [B, H, N, D] (bf16, f16 or fp32; any strides) over the cache, new tokens among its tokens:

        out_i = sum_j softmax_j(scale * q_i.k_j + log_mass[j]) v_j     over j < lengths[b]

    lengths int32 [B]: tokens of each sequence, those of this call's queries included; counts int32 [B] (default N): how many
    of its queries are real; query i stands at place lengths[b] - counts[b] + i, and with `causal` sees no later one.
    H is a multiple of the cache's Hk (head h reads key head h // (H // Hk)); scale (1e-8 to 1e8) defaults to 1 / sqrt(D).  Returns
    [B, H, N, D], token-major in memory where q is; zeros for padding and for queries that attend to nothing (a
    log mass of -inf, or no page, keeps a token out; masses past 1e30 in size count as that, but for -inf).  A query with a channel
    that is not finite, or that sees a mass of NaN, comes out as NaN, unless it attends to nothing.

    Tokens past a length, or past the table (2**30 tokens a sequence at most), are not there and may hold anything, and so may
    those that a mass of -inf keeps out; others must be finite where any query of their sequence can see them.  Stored numbers
    enter exactly (in f16, with many queries, values below 2**-23 to its smallest number, 2**-24).  Sums are fp32; probabilities
    are rounded to a 16-bit type of q where queries are many (more than 64 rows beside a key head, a row being a query of one
    of the key head's heads), else taken to twice its bits (as may be the last 64 of many rows), and to 24 bits in fp32.
    Results are the same bits every time for the same call; which queries stand beside one may change its last bits.  Products
    and sums must lie within fp32's range.  Under bf16 or f16 autocast fp32 q is cast first."""
    _ready(q, cache.data, cache.log_mass, page_table, lengths, counts)
    (q,) = _autocast(q)
    if scale is None:
        scale = 1.0 / math.sqrt(cache.head_dim)
    return torch.ops.vgo.cached_attention(q, cache.data, cache.log_mass, page_table, lengths, counts, bool(causal),
                                          float(scale))
