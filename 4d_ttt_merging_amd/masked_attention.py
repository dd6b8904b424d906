"""Attention under score caps, position biases and masks, with gradients, on gfx950.

`masked_attention` computes, for queries i at position p_i and keys j,

    z_ij = cap * tanh(scale * q_i.k_j / cap) + log_key_mass[j] - slopes[h] * |j - p_i|
           + bucket_table[bucket(j - p_i), h]
    out_i = sum_j softmax_j(z_ij) v_j      over the pairs that attend

(csrc/masked_attention.hip, gradients csrc/masked_attention_grad.hip), and
`relative_position_bias` the table's bias as a dense tensor (csrc/position_bias.hip).  Neither has a
counterpart in the reference, whose attention is unmasked and inference only
(vggt_omega/models/mass_bias_attention.py:85-129); there is no CPU path.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib


@functools.lru_cache(maxsize=None)
def _bucket_starts(buckets: int, max_distance: int, bidirectional: bool) -> tuple[int, ...]:
    """The smallest |distance| of buckets 1, 2, ... of one direction.

    Of the n buckets of a direction (half of them all if bidirectional) the first e = n // 2 hold one
    distance each; the other m = n - e grow with the logarithm up to `max_distance`, from which on
    all distances share the last: d lies in bucket e + floor(m log(d / e) / log(max_distance / e)).
    Taken in whole numbers, d**m >= e**(m - t) * max_distance**t, so no border depends on a
    rounded logarithm."""
    if bidirectional and (buckets < 4 or buckets % 2):
        raise ValueError("a bidirectional bias needs an even number of buckets, 4 at least")
    if buckets < 2 or buckets > 256:
        raise ValueError("a position bias has 2 to 256 buckets")
    n = buckets // 2 if bidirectional else buckets
    if n > 128:
        raise ValueError("a position bias has at most 128 buckets a direction")
    e = n // 2
    m = n - e
    if not e < max_distance <= 1 << 20:
        raise ValueError("max_distance must exceed the distances with a bucket of their own, and not 2**20")
    starts = list(range(1, e + 1))
    for t in range(1, m):
        bound, low, high = e ** (m - t) * max_distance ** t, e, max_distance
        while low < high:
            middle = (low + high) // 2
            if middle ** m >= bound:
                high = middle
            else:
                low = middle + 1
        starts.append(low)
    if starts[-1] > 1024:
        raise ValueError("the last bucket of a position bias must start at a distance of 1024 or less")
    return tuple(starts)


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_key_mass: torch.Tensor | None = None, *,
                     causal: bool = False, prefix_lengths: torch.Tensor | None = None,
                     documents: torch.Tensor | None = None, key_documents: torch.Tensor | None = None,
                     key_lengths: torch.Tensor | None = None, query_starts: torch.Tensor | None = None,
                     score_cap: float | None = None, slopes: torch.Tensor | None = None,
                     bucket_table: torch.Tensor | None = None, bidirectional: bool = True, max_distance: int = 128,
                     scale: float | None = None) -> torch.Tensor:
    """Attention with capped scores, position biases and masks; differentiable in q, k, v, log_key_mass,
    slopes and bucket_table (once, in reverse mode).

    q [B, H, Nq, D], k and v [B, Hk, Nk, D] of one type (bf16, f16 or fp32), D 64 or 128, H a multiple of
    Hk (head h reads key head h // (H // Hk)); any strides, those of a packed projection without a copy.
    Returns [B, H, Nq, D], token-major in memory where q is.  Under bf16 or f16 autocast fp32 operands are
    cast first.

    Position of query i: query_starts[b] + i (int32 [B]; default Nk - Nq, the queries at the keys' end).
    Scores:
      scale         default 1 / sqrt(D); positive
      score_cap     cap * tanh(score / cap); None or 0: none.  Of any size: past 1e15 it leaves scores as they are
      log_key_mass  floating [Nk], added to every score of that key (taken in fp32, not rounded to q's type
                    as `mass_bias_attention` does); -inf keeps a key out, while a type's lowest value is a
                    number: where a row's keys have nothing else it is a mean over them
      slopes        floating [H]: less slopes[h] * distance
      bucket_table  floating [buckets, H]: plus its row for the bucket of the distance, as in
                    `relative_position_bias` (`bidirectional`, `max_distance`)
    A pair attends unless one of these keeps it from it:
      causal          j <= position, or j < prefix_lengths[b] (int32 [B])
      documents       int32 [B, Nq] (and key_documents [B, Nk], default the same): equal and not negative;
                      tiles of 64 keys none of whose documents can match are skipped, so tokens of a document
                      should stand together
      key_lengths     int32 [B]: j < key_lengths[b]
    A query that attends to nothing gives zeros, and no gradient.  Keys past key_lengths and keys of
    negative documents are never read and may hold anything; other keys and values must be finite
    wherever some query of their 64 attends to them.  Few queries (a decoding step: Nq below 32) take the
    heads of one key head together and split the keys over the chip.  Results and gradients are the
    same bits every time.

    Products take probabilities and score gradients rounded to the operands' type; sums are fp32.  A call that
    records a graph divides by the sum of the unrounded probabilities (bf16), and with slopes multiplies what
    rounding took from them too, so its output is not bit for bit that of the same call without one.  For its
    backward it keeps q, k, v, the output, two fp32 numbers a row and, of 16-bit types, as much again as the
    output (what rounding took from it).  Score gradients in f16 lose bits below 2^-14 and are gone below
    2^-25: scale the loss."""
    try:
        _lib.load()
    except _lib.ExtensionUnavailable as error:
        raise RuntimeError(str(error)) from error
    _lib.require_gpu(q, k, v, log_key_mass, slopes, bucket_table, prefix_lengths, documents, key_documents,
                     key_lengths, query_starts)
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be [batch, heads, tokens, channels]")
    if q.shape[-1] not in (64, 128):
        raise ValueError("masked_attention takes 64 or 128 channels a head")
    if q.dtype == torch.float32 and torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        if dtype in (torch.bfloat16, torch.float16):
            q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    if q.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {q.dtype}")
    if prefix_lengths is not None and not causal:
        raise ValueError("prefix_lengths go with causal=True")
    if documents is None and key_documents is not None:
        raise ValueError("key_documents need the queries' documents")
    if documents is not None and key_documents is None:
        if q.shape[2] != k.shape[2]:
            raise ValueError("queries beside other keys need key_documents")
        key_documents = documents
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if not 0.0 < scale < math.inf:
        raise ValueError("the scale must be positive and finite")
    cap = 0.0 if score_cap is None else float(score_cap)
    if not 0.0 <= cap < math.inf:
        raise ValueError("the score cap must be finite and not negative")
    starts = ()
    if bucket_table is not None:
        if bucket_table.ndim != 2:
            raise ValueError("bucket_table must be [buckets, heads]")
        starts = _bucket_starts(bucket_table.shape[0], int(max_distance), bool(bidirectional))
    if log_key_mass is not None:
        log_key_mass = log_key_mass.reshape(-1)
    return torch.ops.vgo.masked_attention(
        q, k, v, log_key_mass, slopes, bucket_table, prefix_lengths, documents, key_documents, key_lengths,
        query_starts, float(scale), cap, starts, bool(bidirectional), bool(causal), False)[0]


def relative_position_bias(table: torch.Tensor, n_query: int, n_key: int, *, query_start: int | None = None,
                           bidirectional: bool = True, max_distance: int = 128) -> torch.Tensor:
    """The bias of `masked_attention`'s bucket_table as a tensor [heads, n_query, n_key] of the table's type:
    table[bucket(j - position of i), head], the position of query i being query_start + i (default
    n_key - n_query).  Differentiable in the table [buckets, heads] (its gradient is summed in fp32).

    Buckets: half of them for keys behind the query, half for keys ahead (bidirectional), or all for keys
    behind (keys ahead then share bucket 0 with distance 0).  Half of a direction's buckets hold one
    distance each, the others grow with the logarithm up to `max_distance`.  Where it only ever is added to
    scores, give the table to `masked_attention`, which never writes the tensor out."""
    try:
        _lib.load()
    except _lib.ExtensionUnavailable as error:
        raise RuntimeError(str(error)) from error
    _lib.require_gpu(table)
    if table.ndim != 2:
        raise ValueError("the table must be [buckets, heads]")
    if table.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {table.dtype}")
    if n_query < 0 or n_key < 0:
        raise ValueError("negative size")
    starts = _bucket_starts(table.shape[0], int(max_distance), bool(bidirectional))
    start = n_key - n_query if query_start is None else int(query_start)
    return torch.ops.vgo.position_bias(table, n_query, n_key, start, starts, bool(bidirectional))
