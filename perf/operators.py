"""Masked attention with position biases, its gradients and its single-token form, and the
relative position bias by buckets, as cases that can be timed and checked.

`own` selects what `run` does: the operators in plain torch operations (32 bits, rounded once at the
end), or the package's entry points `masked_attention` and `relative_position_bias`.  Heads, widths
and lengths are those of the aggregator (16 heads of 64 channels, 1,029 tokens per frame of
512 x 512, 261 of a small one, 4 to 32 frames), with grouped key heads and 128 channels beside them.
"""
from __future__ import annotations

import functools
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
# What a case leaves out.
DEFAULTS = dict(batch=1, heads=16, kv_heads=16, dim=64, causal=False, prefix=0, doc=0, ragged=0, cap=0.0,
                bias="none", buckets=32, distance=128, mass=False, gain=1.0)


# ------------------------------------------------------------------ cases ----
def listed() -> list[dict]:
    return [
        # A layer of one small frame with capped scores: over in microseconds, launches count.
        dict(name="forward_261_cap_bf16", kind="forward", dtype="bf16", nq=261, nk=261, causal=True, cap=30.0, gain=2.0),
        # 16 ragged frames packed in one row, each attending to itself (a document mask), padding behind.
        dict(name="forward_frames_bf16", kind="forward", dtype="bf16", nq=16464, nk=16464, doc=1029),
        # The same tokens attending over all frames so far, merged keys with their masses, capped.
        dict(name="forward_causal_cap_bf16", kind="forward", dtype="bf16", nq=16464, nk=16464, causal=True, cap=50.0,
             mass=True, gain=2.0),
        # A prefix of frames that see each other, then causal tokens; 128 channels, 4 key heads.
        dict(name="forward_prefix_128_f16", kind="forward", dtype="f16", nq=4111, nk=4111, causal=True, prefix=1029,
             heads=16, kv_heads=4, dim=128),
        # A training step's attention: two sequences of two frames, causal, capped.
        dict(name="train_causal_cap_bf16", kind="train", dtype="bf16", batch=2, nq=2058, nk=2058, causal=True, cap=30.0,
             gain=2.0),
        # The same with a learned bucket bias over ragged packed documents, grouped key heads.
        dict(name="train_buckets_bf16", kind="train", dtype="bf16", batch=2, nq=1029, nk=1029, doc=261, kv_heads=4,
             bias="buckets"),
        # The long one: eight frames, prefix mask, 128 channels, masses with their gradient.
        dict(name="train_long_128_bf16", kind="train", dtype="bf16", nq=8232, nk=8232, causal=True, prefix=2058, dim=128,
             heads=16, kv_heads=8, mass=True),
        # A small fp32 training step with slopes and bucket table of an unmerged and a merged length.
        dict(name="train_slopes_fp32", kind="train", dtype="fp32", nq=522, nk=1044, bias="slopes", mass=True, heads=8,
             kv_heads=8),
        # One new token of one sequence: latency alone.
        dict(name="token_1_bf16", kind="forward", dtype="bf16", nq=1, nk=1044, bias="slopes", kv_heads=4),
        # One new token each of 32 sequences over caches of up to 32 frames, ragged lengths, capped.
        dict(name="token_32_bf16", kind="forward", dtype="bf16", batch=32, nq=1, nk=32928, ragged=1, cap=30.0, kv_heads=4,
             gain=2.0),
        # The dense bias of a two-frame layer and the gradient of its table.
        dict(name="bias_2058_bf16", kind="bias", dtype="bf16", nq=2058, nk=2058),
        dict(name="bias_261_fp32", kind="bias", dtype="fp32", nq=261, nk=1044),
    ]


def _log_uniform(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["forward", "forward", "train", "train", "token", "bias"])
    dtype = rng.choice(["bf16", "bf16", "f16", "fp32"])
    heads = rng.choice([8, 16])
    if kind == "bias":
        return dict(kind=kind, dtype=dtype, heads=heads, nq=_log_uniform(rng, 1, 2058), nk=_log_uniform(rng, 200, 2058),
                    buckets=rng.choice([16, 32, 64]), distance=rng.choice([64, 128, 500]))
    case = dict(kind="train" if kind == "train" else "forward", dtype=dtype, heads=heads,
                kv_heads=rng.choice([heads, heads, heads // 4]), dim=rng.choice([64, 64, 128]),
                cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice(["none", "none", "slopes", "buckets"]),
                gain=rng.choice([1.0, 2.0]))
    if kind == "token":
        return dict(case, batch=rng.randint(1, 32), nq=rng.choice([1, 1, 2, 4]), nk=_log_uniform(rng, 500, 32928),
                    ragged=1)
    n = _log_uniform(rng, 60, {"forward": 10000, "train": 5000}[kind] // (4 if dtype == "fp32" else 1))
    mask = rng.choice(["none", "causal", "prefix", "doc", "causal doc"])
    case.update(batch=rng.choice([1, 1, 2]), nq=n, nk=n, causal=mask.startswith(("causal", "prefix")),
                prefix=n // rng.randint(2, 6) if mask == "prefix" else 0,
                doc=max(16, n // rng.randint(2, 12)) if "doc" in mask else 0, mass=rng.random() < 0.3)
    if mask == "none" and rng.random() < 0.5:  # queries beside merged keys
        case["nk"] = max(16, int(n * rng.uniform(0.25, 1.0)))
    return case


# ----------------------------------------------------------------- inputs ----
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case: dict, seed: int):
    c = {**DEFAULTS, **case}
    g = _generator(seed)
    dtype = DTYPES[c["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if c["kind"] == "bias":
        return dict(c, table=randn(c["buckets"], c["heads"]).requires_grad_(),
                    grad=randn(c["heads"], c["nq"], c["nk"]))
    train = c["kind"] == "train"
    b, nq, nk = c["batch"], c["nq"], c["nk"]
    # Token-major rows as a packed projection gives them, seen head-major.
    q = randn(b, nq, c["heads"], c["dim"], scale=c["gain"]).transpose(1, 2)
    k = randn(b, nk, c["kv_heads"], c["dim"]).transpose(1, 2)
    v = randn(b, nk, c["kv_heads"], c["dim"]).transpose(1, 2)
    state = dict(c, q=q, k=k, v=v, mass_log=None, slopes=None, table=None, prefix_lengths=None, documents=None,
                 key_lengths=None, query_starts=None)
    if c["mass"]:
        state["mass_log"] = torch.randint(1, 9, (nk,), generator=g, device="cuda").float().log().to(dtype)
    if c["bias"] == "slopes":
        state["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["heads"] + 1, device="cuda") / c["heads"]).to(dtype)
    if c["bias"] == "buckets":
        state["table"] = randn(c["buckets"], c["heads"], scale=0.5)
    if c["prefix"]:
        state["prefix_lengths"] = torch.full((b,), c["prefix"], dtype=torch.int32, device="cuda")
    if c["doc"]:
        # Segments around the given length, at places of their own for each sequence; the last few rows are padding.
        cuts = torch.rand(b, nq, generator=g, device="cuda") < 1.0 / c["doc"]
        documents = cuts.cumsum(1).to(torch.int32)
        documents[:, nq - nq // 50:] = -1
        state["documents"] = documents
    if c["ragged"]:
        lengths = torch.randint(max(1, nk // 4), nk + 1, (b,), generator=g, device="cuda").to(torch.int32)
        state["key_lengths"] = lengths
        state["query_starts"] = lengths - nq
    if train:
        for name in ("q", "k", "v", "mass_log", "slopes", "table"):
            if state[name] is not None:
                state[name].requires_grad_()
        state["grad"] = randn(b, nq, c["heads"], c["dim"]).transpose(1, 2)
    return state


# ------------------------------------------------------------- plain form ----
@functools.lru_cache(maxsize=None)
def _bucket_starts(buckets: int, distance: int, bidirectional: bool) -> tuple[int, ...]:
    """Smallest |distance| of buckets 1, 2, ... of one direction: the first half hold one distance
    each, the others grow with the logarithm up to `distance`.  In whole numbers: bucket e + t
    starts at the smallest n with (n / e)^m >= (distance / e)^t."""
    per = buckets // 2 if bidirectional else buckets
    e = per // 2
    m = per - e
    grown = [next(n for n in range(e, distance + 1) if n ** m >= e ** (m - t) * distance ** t) for t in range(1, m)]
    return tuple([*range(1, e + 1), *grown])


def _buckets(relative: torch.Tensor, buckets: int, distance: int) -> torch.Tensor:
    """Bucket of every key position less query position, both directions."""
    starts = torch.tensor(_bucket_starts(buckets, distance, True), device=relative.device)
    return torch.bucketize(relative.abs(), starts, right=True) + (relative > 0) * (buckets // 2)


def _relative(s) -> torch.Tensor:
    """Key position less query position [b or 1, nq, nk]."""
    starts = s["query_starts"]
    starts = torch.tensor([s["nk"] - s["nq"]], device="cuda") if starts is None else starts.long()
    position = starts[:, None] + torch.arange(s["nq"], device="cuda")
    return torch.arange(s["nk"], device="cuda") - position[:, :, None]


def _allowed(s, relative: torch.Tensor) -> torch.Tensor | None:
    """Pairs that attend [b or 1, nq, nk], or None where all do."""
    j = torch.arange(s["nk"], device="cuda")
    ok = None
    if s["causal"]:
        ok = relative <= 0
        if s["prefix_lengths"] is not None:
            ok = ok | (j < s["prefix_lengths"][:, None, None])
    if s["documents"] is not None:
        d = s["documents"]
        same = (d[:, :, None] == d[:, None, :]) & (d[:, :, None] >= 0)
        ok = same if ok is None else ok & same
    if s["key_lengths"] is not None:
        inside = j < s["key_lengths"][:, None, None]
        ok = inside if ok is None else ok & inside
    return ok


def _plain_attention(s) -> torch.Tensor:
    b, h, hk, nq, nk, d = s["batch"], s["heads"], s["kv_heads"], s["nq"], s["nk"], s["dim"]
    q = s["q"].float().reshape(b, hk, h // hk * nq, d)
    k, v = s["k"].float(), s["v"].float()
    scores = (q @ k.transpose(-1, -2) * d ** -0.5).view(b, h, nq, nk)
    if s["cap"]:
        scores = torch.tanh(scores / s["cap"]) * s["cap"]
    if s["mass_log"] is not None:
        scores = scores + s["mass_log"].float()
    relative = _relative(s)
    if s["slopes"] is not None:
        scores = scores - s["slopes"].float()[:, None, None] * relative.abs().float()[:, None]
    if s["table"] is not None:
        # A product with the 0/1 matrix of the buckets: its gradient is a product too, not a scatter.
        held = _buckets(relative, s["buckets"], s["distance"])[..., None] == torch.arange(s["buckets"], device="cuda")
        scores = scores + (held.float() @ s["table"].float()).permute(0, 3, 1, 2)
    ok = _allowed(s, relative)
    if ok is not None:
        scores = scores.masked_fill(~ok[:, None], -math.inf)
    peak = scores.detach().amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(peak == -math.inf, 0.0, peak))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p.view(b, hk, h // hk * nq, nk) @ v
    return out.view(b, h, nq, d).to(s["q"].dtype)


def _plain_bias(s):
    relative = torch.arange(s["nk"], device="cuda") - (s["nk"] - s["nq"] + torch.arange(s["nq"], device="cuda"))[:, None]
    bias = s["table"].detach()[_buckets(relative, s["buckets"], s["distance"])].permute(2, 0, 1).contiguous()
    # Rows of the gradient sheared until every distance is a column, summed; then the distances of each bucket.
    h, nq, nk = s["grad"].shape
    wide = torch.nn.functional.pad(s["grad"].float().flip(1), (0, nq)).view(h, -1)[:, :nq * (nk + nq - 1)]
    by_distance = wide.view(h, nq, nk + nq - 1).sum(1)
    distance = torch.arange(nk + nq - 1, device="cuda") - (nq - 1) - (nk - nq)
    bucket = _buckets(distance, s["buckets"], s["distance"])
    held = (bucket[:, None] == torch.arange(s["buckets"], device="cuda")).double()
    return bias, (by_distance.double() @ held).t().to(s["table"].dtype).contiguous()


# ----------------------------------------------------------------- passes ----
@functools.lru_cache(maxsize=1)
def _vgo():
    return importlib.import_module("4d_ttt_merging_amd")


def _own_attention(s) -> torch.Tensor:
    return _vgo().masked_attention(
        s["q"], s["k"], s["v"], s["mass_log"], causal=s["causal"], prefix_lengths=s["prefix_lengths"],
        documents=s["documents"], key_lengths=s["key_lengths"], query_starts=s["query_starts"],
        score_cap=s["cap"] or None, slopes=s["slopes"], bucket_table=s["table"], max_distance=s["distance"])


def run(s):
    if s["kind"] == "bias":
        if not own:
            return dict(zip(("bias", "table"), _plain_bias(s)))
        bias = _vgo().relative_position_bias(s["table"], s["nq"], s["nk"], max_distance=s["distance"])
        return dict(bias=bias.detach(), table=torch.autograd.grad(bias, s["table"], s["grad"])[0])
    attention = _own_attention if own else _plain_attention
    if s["kind"] == "forward":
        with torch.no_grad():
            return attention(s)
    out = attention(s)
    names = [n for n in ("q", "k", "v", "mass_log", "slopes", "table") if s[n] is not None]
    grads = torch.autograd.grad(out, [s[n] for n in names], s["grad"])
    return dict(zip(names, grads), out=out.detach())


# ------------------------------------------------------------ work, exact ----
def _pairs(c: dict) -> float:
    """Pairs that attend in one sequence and head, on average over the inputs."""
    nq, nk = c["nq"], c["nk"]
    if c["doc"]:
        # A token's document is twice the mean length long on average, less at the ends of the row.
        return nq * min(nk, 2 * c["doc"] * (1 - min(0.5, c["doc"] / nq))) * (0.5 if c["causal"] else 1.0)
    keys = nk * (0.625 if c["ragged"] else 1.0)
    if c["causal"]:
        return nq * keys - nq * (nq - 1) / 2 + c["prefix"] * (c["prefix"] - 1) / 2
    return nq * keys


def work(case: dict) -> dict:
    c = {**DEFAULTS, **case}
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "bias":
        return {"bytes": 2 * size * c["heads"] * c["nq"] * c["nk"], "flops": c["heads"] * c["nq"] * c["nk"]}
    keys = c["nk"] * (0.625 if c["ragged"] else 1.0)
    rows = c["batch"] * c["dim"] * size
    q, kv = rows * c["heads"] * c["nq"], rows * c["kv_heads"] * keys
    product = 2.0 * c["batch"] * c["heads"] * c["dim"] * _pairs(c)
    if c["kind"] == "forward":
        return {"bytes": int(2 * q + 2 * kv), "flops": int(2 * product)}
    return {"bytes": int(4 * q + 4 * kv), "flops": int(7 * product)}


def exact(case: dict, seed: int):
    """64 bits, one key head at a time, gradients by their formulas."""
    s = prepare(case, seed)
    if s["kind"] == "bias":
        table, grad = s["table"].detach().double(), s["grad"].double()
        rel = torch.arange(s["nk"], device="cuda")[None] - torch.arange(s["nk"] - s["nq"], s["nk"], device="cuda")[:, None]
        bucket = _exact_bucket(rel, s["buckets"], s["distance"])
        sums = torch.zeros(s["buckets"], s["heads"], dtype=torch.float64, device="cuda")
        for t in range(s["buckets"]):
            sums[t] = (grad * (bucket == t)).sum((1, 2))
        return dict(bias=table[bucket].permute(2, 0, 1), table=sums)
    b, h, hk, nq, nk, d = s["batch"], s["heads"], s["kv_heads"], s["nq"], s["nk"], s["dim"]
    if b * h * nq * nk > 6e9:
        return None
    group, f64, train = h // hk, torch.float64, s["kind"] == "train"
    scale, cap = 1.0 / math.sqrt(d), s["cap"]
    wide = {n: None if s[n] is None else s[n].detach().to(f64) for n in ("q", "k", "v", "mass_log", "slopes", "table")}
    result = dict(out=torch.zeros(b, h, nq, d, dtype=f64, device="cuda"))
    if train:
        result.update({n: torch.zeros_like(t) for n, t in wide.items() if t is not None})
    j = torch.arange(nk, device="cuda")
    for i in range(b):
        start = nk - nq if s["query_starts"] is None else int(s["query_starts"][i])
        gap = j[None, :] - (start + torch.arange(nq, device="cuda"))[:, None]
        mask = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if s["key_lengths"] is not None:
            mask &= j < int(s["key_lengths"][i])
        if s["causal"]:
            mask &= (gap <= 0) | (j < s["prefix"])
        if s["documents"] is not None:
            row = s["documents"][i]
            mask &= (row[:, None] == row[None, :]) & (row >= 0)[:, None]
        bucket = None if s["table"] is None else _exact_bucket(gap, s["buckets"], s["distance"])
        for head in range(h):
            kv = head // group
            q, k, v = wide["q"][i, head], wide["k"][i, kv], wide["v"][i, kv]
            z = q @ k.T * scale
            bend = None
            if cap:
                bend = torch.tanh(z / cap)
                z = cap * bend
            if wide["mass_log"] is not None:
                z = z + wide["mass_log"]
            if wide["slopes"] is not None:
                z = z - wide["slopes"][head] * gap.abs()
            if bucket is not None:
                z = z + wide["table"][:, head][bucket]
            z = torch.where(mask, z, -math.inf)
            weight = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            o = weight @ v
            result["out"][i, head] = o
            if not train:
                continue
            go = s["grad"][i, head].to(f64)
            result["v"][i, kv] += weight.T @ go
            dz = weight * (go @ v.T - (go * o).sum(-1, keepdim=True))
            if wide["mass_log"] is not None:
                result["mass_log"] += dz.sum(0)
            if wide["slopes"] is not None:
                result["slopes"][head] -= (dz * gap.abs()).sum()
            if bucket is not None:
                for t in range(s["buckets"]):
                    result["table"][t, head] += dz[bucket == t].sum()
            if bend is not None:
                dz = dz * (1 - bend * bend)
            result["q"][i, head] = dz @ k * scale
            result["k"][i, kv] += dz.T @ q * scale
    return result if train else result["out"]


def _exact_bucket(gap: torch.Tensor, buckets: int, distance: int) -> torch.Tensor:
    """Bucket of each gap from the definition: half + floor(log(n / half) / log(distance / half) * half) beyond the
    first half, in 64 bits with a nudge that only moves what lies on a border."""
    per = buckets // 2
    half = per // 2
    n = gap.abs()
    grown = torch.log(n.clamp(min=1).double() / half) / math.log(distance / half) * (per - half)
    far = (half + torch.floor(grown + 1e-9).long()).clamp(max=per - 1)
    return torch.where(n < half, n, far) + per * (gap > 0)
