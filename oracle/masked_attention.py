"""Masked attention with position biases and its gradients in 64 bits, with error bounds.

Written from the definition (4d_ttt_merging_amd/masked_attention.py states it): scores, masks and
gradients by their formulas, one (batch, head) at a time.  `bounds` gives, element by element, how far
a kernel may be off that keeps sums in fp32 and rounds probabilities, score gradients and results to the
inputs' type: half a step each, u = eps / 2.
"""
from __future__ import annotations

import math

import torch


def bucket(distance: torch.Tensor, buckets: int, max_distance: int, bidirectional: bool) -> torch.Tensor:
    """Bucket of each signed distance, borders compared in whole numbers."""
    n = buckets // 2 if bidirectional else buckets
    e = n // 2
    m = n - e

    def one(d: int) -> int:
        side = n if bidirectional and d > 0 else 0
        d = abs(d) if bidirectional else max(-d, 0)
        if d < e:
            return side + d
        t = 0
        while t + 1 < m and d ** m >= e ** (m - t - 1) * max_distance ** (t + 1):
            t += 1
        return side + e + t

    values = {int(d): one(int(d)) for d in distance.unique()}
    return distance.clone().apply_(lambda d: values[int(d)])


def relative_position_bias(table, n_query, n_key, *, query_start=None, bidirectional=True, max_distance=128):
    start = n_key - n_query if query_start is None else query_start
    gap = torch.arange(n_key) - (start + torch.arange(n_query))[:, None]
    return table[bucket(gap, table.shape[0], max_distance, bidirectional)].permute(2, 0, 1)


def attention(q, k, v, log_key_mass=None, *, grad=None, causal=False, prefix_lengths=None, documents=None,
              key_documents=None, key_lengths=None, query_starts=None, score_cap=None, slopes=None, bucket_table=None,
              bidirectional=True, max_distance=128, scale=None, dtype=None):
    """(results, bounds): dicts of float64 tensors `out` and, with `grad` (the gradient of out), `q`, `k`, `v` and
    those of log_key_mass, slopes and bucket_table.  `dtype`: the type the bounds are for (default q's)."""
    dtype = dtype or q.dtype
    u = torch.finfo(dtype).eps / 2
    u32 = 2.0 ** -24
    b, h, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    wide = [None if t is None else t.detach().double().cpu() for t in (q, k, v, log_key_mass, slopes, bucket_table, grad)]
    q, k, v, mass, slopes, table, grad = wide
    whole = [None if t is None else t.cpu().long() for t in
             (prefix_lengths, documents, documents if key_documents is None else key_documents, key_lengths, query_starts)]
    prefix, qdoc, kdoc, lengths, starts = whole
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    j = torch.arange(nk)
    res = dict(out=torch.zeros_like(q))
    if grad is not None:
        res.update(q=torch.zeros_like(q), k=torch.zeros_like(k), v=torch.zeros_like(v))
        res.update({n: torch.zeros_like(t) for n, t in (("log_key_mass", mass), ("slopes", slopes), ("bucket_table", table))
                    if t is not None})
    err = {n: torch.zeros_like(t) for n, t in res.items()}
    for i in range(b):
        pos = (nk - nq if starts is None else int(starts[i])) + torch.arange(nq)
        gap = j - pos[:, None]
        ok = torch.ones(nq, nk, dtype=torch.bool)
        dead = torch.zeros(nk, dtype=torch.bool)  # keys nothing may read
        if lengths is not None:
            dead |= j >= int(lengths[i])
        if kdoc is not None:
            dead |= kdoc[i] < 0
            ok &= qdoc[i][:, None] == kdoc[i]
        if causal:
            seen = gap <= 0
            ok &= seen if prefix is None else seen | (j < int(prefix[i]))
        ok &= ~dead
        which = None if table is None else bucket(gap, table.shape[0], max_distance, bidirectional)
        alive = ok.any(1, keepdim=True)
        for head in range(h):
            kv = head // (h // hk)
            ki, vi = (t[i, kv].masked_fill(dead[:, None], 0.0) for t in (k, v))
            qi = q[i, head].masked_fill(~alive, 0.0)
            raw = qi @ ki.T * scale
            z, bend = raw, torch.ones_like(raw)
            if score_cap:
                t = torch.tanh(raw / score_cap)
                z, bend = t * score_cap, 1 - t * t
            if mass is not None:
                z = z + mass
            if slopes is not None:
                z = z - slopes[head] * gap.abs()
            if table is not None:
                z = z + table[:, head][which]
            live = ok & (z != -math.inf)
            zm = torch.where(live, z, -math.inf)
            top = zm.amax(1, keepdim=True) if nk else torch.full((nq, 1), -math.inf)
            e = torch.exp(zm - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(1, keepdim=True)
            p = e / torch.where(total == 0, 1.0, total)
            out = p @ vi
            res["out"][i, head] = out
            # Relative error of p in fp32: a dot product of d terms (each addition half a step of the sum of
            # magnitudes), a few roundings of the score and of exp2's argument, and the row sum of nk terms.
            if nk:
                dots = (qi.abs() @ ki.abs().T * scale).max()
                size = torch.where(live, z.abs(), 0.0).max()
                if slopes is not None:
                    size = size + slopes[head].abs() * gap.abs().max()
                kappa = float(2 * ((d + 4) * dots + 8 * size + 12) + nk) * u32
            else:
                kappa = 0.0
            rounded = 0.0 if dtype == torch.float32 else u
            a = p @ vi.abs()
            err["out"][i, head] = (rounded + kappa) * a + u * out.abs()
            if grad is None:
                continue
            go = grad[i, head].masked_fill(~(live.any(1, keepdim=True)), 0.0)
            qg = qi.masked_fill(~(live.any(1, keepdim=True)), 0.0)
            dp = go @ vi.T
            delta = (go * out).sum(1, keepdim=True)
            dz = p * (dp - delta)
            ds = dz * bend
            res["v"][i, kv] += p.T @ go
            res["q"][i, head] = ds @ ki * scale
            res["k"][i, kv] += ds.T @ qg * scale
            # delta comes from the rounded out; dP, delta and p each in fp32.
            d_delta = (go.abs() * err["out"][i, head]).sum(1, keepdim=True) + (d + 4) * u32 * (go.abs() * out.abs()).sum(1, keepdim=True)
            size = go.abs() @ vi.abs().T + (go.abs() * a).sum(1, keepdim=True)
            e_dz = p * d_delta + (kappa + (d + 4) * u32) * p * size
            # cap' = 1 - t^2 carries the score's error: d(cap')/d(raw) = -2 t cap' / cap, and 2^-22 of rounding.
            e_ds = rounded * ds.abs() + e_dz * bend.clamp(max=1.0)
            if score_cap:
                e_ds = e_ds + (p * size) * (2.0 ** -21 + 2 * kappa / score_cap)
            long = (nq * (h // hk) + nk) * u32
            err["v"][i, kv] += (rounded + kappa + long) * (p.T @ go.abs())
            err["q"][i, head] = ((e_ds + long * ds.abs()) @ ki.abs()) * scale + u * res["q"][i, head].abs()
            err["k"][i, kv] += ((e_ds + long * ds.abs()).T @ qg.abs()) * scale
            far = (b * h * nq + nk) * u32
            if mass is not None:
                res["log_key_mass"] += dz.sum(0)
                err["log_key_mass"] += (e_dz + far * dz.abs()).sum(0)
            if slopes is not None:
                res["slopes"][head] -= (dz * gap.abs()).sum()
                err["slopes"][head] += ((e_dz + far * dz.abs()) * gap.abs()).sum()
            if table is not None:
                res["bucket_table"][:, head] += torch.zeros(table.shape[0], dtype=torch.float64).index_add_(0, which.flatten(), dz.flatten())
                err["bucket_table"][:, head] += torch.zeros(table.shape[0], dtype=torch.float64).index_add_(
                    0, which.flatten(), (e_dz + far * dz.abs()).flatten())
    if grad is not None:
        for n in ("k", "v"):
            err[n] += u * res[n].abs()
    return res, err
