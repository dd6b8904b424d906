"""The paged cache of keys and values in 4 bits -- appending with the position rotation, reading tokens back,
attention over it -- as cases that can be timed and checked.

`own` selects what `run` does: the operators in plain torch operations (32 bits, 64 for the rotation and the
choice of codes; rounded once at the end), or the package's entry points `cache_append`, `cache_read` and
`cached_attention`.  Heads, widths and lengths are those of the aggregator (16 heads of 64 channels, 1,029 tokens
per frame of 512 x 512, 261 of a small one, 4 to 32 frames), with grouped key heads and 128 channels beside them.

The cache: uint8 [pages, key heads, page_size / 32, 34 * dim], blocks of 32 tokens, each
    keys' codes   [32 tokens][dim / 2]           byte c: channel 2c in its low half, 2c + 1 in its high half
    values' codes [4][dim / 2][8 tokens]         tokens 8g .. 8g + 7 of a channel pair side by side
    keys' scales  [32 tokens][dim / 32]          2^(byte - 127), one for 32 channels of a token; 255: NaN
    values' scales [4][dim / 32][8 tokens]
and a code s.m of 4 bits stands for the m-th of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign.
"""
from __future__ import annotations

import functools
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# What a case leaves out.  nq: new tokens of a sequence (those of the longest, if ragged); nk: tokens of the longest
# sequence with them; table: rows of the rotation's tables, 0: none; special: tokens in front that are not rotated.
DEFAULTS = dict(batch=1, heads=16, kv_heads=16, dim=64, page=64, ragged=False, mass=False, table=0, special=0,
                causal=False, gain=1.0)


# ------------------------------------------------------------------ cases ----
def listed() -> list[dict]:
    return [
        # One new token of one sequence: latency alone.
        dict(name="append_1_bf16", kind="append", dtype="bf16", nq=1, nk=1044, kv_heads=4, table=2048),
        # One new token each of 32 sequences, at places of their own.
        dict(name="append_32_f16", kind="append", dtype="f16", batch=32, nq=1, nk=8232, kv_heads=4, dim=128, table=8232,
             ragged=True),
        # The two halves of a small merged frame in fp32, behind an odd number of tokens.
        dict(name="append_522_fp32", kind="append", dtype="fp32", batch=2, nq=261, nk=522, heads=8, kv_heads=8, page=32,
             table=256, special=5, mass=True),
        # A frame: 5 special tokens that are not rotated, 1,024 patches at their places in the frame, their masses.
        dict(name="append_frame_bf16", kind="append", dtype="bf16", nq=1029, nk=16464, table=1024, special=5, mass=True),
        # Prompts of four scenes, 8 frames at most, ragged.
        dict(name="append_prompts_bf16", kind="append", dtype="bf16", batch=4, nq=8232, nk=8232, table=8232, page=128,
             ragged=True),
        # One new token of one sequence over four small frames: latency alone.
        dict(name="token_1_bf16", kind="attend", dtype="bf16", nq=1, nk=1044, kv_heads=4, gain=2.0),
        # One new token each of 32 sequences over up to 32 frames: the cache's bytes.
        dict(name="token_32_bf16", kind="attend", dtype="bf16", batch=32, nq=1, nk=32928, kv_heads=4, ragged=True, gain=2.0),
        # Four guessed tokens each of 8 sequences, every head its own keys, 128 channels.
        dict(name="guess_4_128_f16", kind="attend", dtype="f16", batch=8, nq=4, nk=16464, heads=16, kv_heads=16, dim=128,
             causal=True, ragged=True),
        # A new frame against all frames so far, itself among them; merged keys with their masses.
        dict(name="frame_bf16", kind="attend", dtype="bf16", nq=1029, nk=32928, mass=True, gain=2.0),
        # Two frames each of two sequences, causal, 128 channels, grouped key heads: the long one.
        dict(name="chunk_128_bf16", kind="attend", dtype="bf16", batch=2, nq=2058, nk=16464, kv_heads=4, dim=128, page=128,
             causal=True, ragged=True),
        # Prompts of three scenes from their start, ragged.
        dict(name="prompts_f16", kind="attend", dtype="f16", batch=3, nq=4116, nk=4116, kv_heads=4, causal=True, ragged=True),
        # A small frame over four of them in fp32.
        dict(name="frame_261_fp32", kind="attend", dtype="fp32", nq=261, nk=1044, heads=8, kv_heads=8, page=32, mass=True),
    ]


def _log_uniform(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "token", "chunk", "chunk"])
    heads = rng.choice([8, 16])
    case = dict(kind="attend", dtype=rng.choice(["bf16", "bf16", "f16", "fp32"]), heads=heads,
                kv_heads=rng.choice([heads, heads, heads // 4, 2]), dim=rng.choice([64, 64, 128]),
                page=rng.choice([32, 64, 64, 128, 256]), mass=rng.random() < 0.3, gain=rng.choice([1.0, 2.0]))
    if kind == "token":
        nk = _log_uniform(rng, 200, 32928)
        return dict(case, batch=rng.randint(1, 16 if case["dim"] == 128 else 32) if nk < 9000 or case["kv_heads"] < 8 else
                    rng.randint(1, 8), nq=rng.choice([1, 1, 2, 5, 8]), nk=nk, causal=rng.random() < 0.7, ragged=rng.random() < 0.7)
    if kind == "append":
        batch = rng.choice([1, 2, 5, 32])
        nq = _log_uniform(rng, 1, 16464 / batch / (2 if case["dim"] == 128 else 1))
        special = rng.choice([0, 0, 1, 5])
        return dict(case, kind="append", batch=batch, nq=nq, nk=nq + _log_uniform(rng, 1, 8000), special=min(special, nq),
                    table=rng.choice([0, 1024, 32928]), ragged=rng.random() < 0.6)
    nq = _log_uniform(rng, 9, 2058 if case["dtype"] != "fp32" else 1029)
    return dict(case, batch=rng.choice([1, 1, 2, 3]), nq=nq, nk=nq + _log_uniform(rng, 1, 12000 if case["dtype"] != "fp32" else 3000),
                causal=rng.random() < 0.6, ragged=rng.random() < 0.5)


# ----------------------------------------------------------------- format ----
def _quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [..., dim] and scale bytes [..., dim / 32] of values.  A block's scale is the smallest power of two, from
    2^-125 to 2^125, of which 7 are at least its largest value: no value is off by more than the scale."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    broken = ~torch.isfinite(top)
    fraction, exponent = torch.frexp(torch.where(broken, 1.0, top))  # top = fraction 2^exponent, 1/2 <= fraction < 1
    e = (exponent - 3 + (fraction > 0.875)).masked_fill(top == 0, -125).clamp(-125, 125)
    y = torch.ldexp(torch.where(broken, 0.0, blocks), -e)
    size = y.abs()
    code = torch.zeros_like(e).expand(y.shape)
    for i in range(7):  # past the middle of two neighbours, or on it where the upper one is the even one
        middle = (LEVELS[i] + LEVELS[i + 1]) / 2
        code = code + (size >= middle if i % 2 else size > middle)
    code = code + 8 * (y < 0)
    return code.flatten(-2).to(torch.uint8), torch.where(broken, 255, e + 127).squeeze(-1).to(torch.uint8)


def _numbers(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 values [..., dim] of codes and scale bytes."""
    levels = torch.tensor([*LEVELS, *(-v for v in LEVELS)], device=codes.device)
    scale = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (levels[codes.int()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _packed(kc, ks, vc, vs) -> torch.Tensor:
    """Blocks uint8 [..., 34 dim] of codes [..., 32, dim] and scale bytes [..., 32, dim / 32]."""
    pair = lambda c: c[..., 0::2] | c[..., 1::2] << 4
    groups = lambda t: t.unflatten(-2, (4, 8)).transpose(-1, -2).flatten(-3)
    return torch.cat([pair(kc).flatten(-2), groups(pair(vc)), ks.flatten(-2), groups(vs)], -1)


def _unpacked(blocks: torch.Tensor, dim: int):
    """(kc, ks, vc, vs) of _packed."""
    kc, vc, ks, vs = blocks.split([16 * dim, 16 * dim, dim, dim], -1)
    halves = lambda t: torch.stack([t & 15, t >> 4], -1).flatten(-2)
    tokens = lambda t: t.unflatten(-1, (4, -1, 8)).transpose(-1, -2).flatten(-3, -2)
    return (halves(kc.unflatten(-1, (32, -1))), ks.unflatten(-1, (32, -1)), halves(tokens(vc)), tokens(vs))


# ----------------------------------------------------------------- inputs ----
def prepare(case: dict, seed: int):
    c = {**DEFAULTS, **case}
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    b, h, hk, d, nq, nk, page = (c[n] for n in ("batch", "heads", "kv_heads", "dim", "nq", "nk", "page"))

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def randint(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda").to(torch.int32)

    # Tokens of a sequence with its new ones, and how many of those are new.
    lengths = torch.full((b,), nk, dtype=torch.int32, device="cuda")
    counts = torch.full((b,), nq, dtype=torch.int32, device="cuda")
    if c["ragged"]:
        if nq > 8:
            counts = randint(max(1, nq // 2), nq + 1, (b,))
        lengths = torch.maximum(randint(max(1, nk // 4), nk + 1, (b,)), counts)
    starts = lengths - counts
    # Pages in no order, as many for each sequence as the longest takes; unused ones are -1.
    per = -(-nk // page)
    table = torch.randperm(b * per + 3, generator=g, device="cuda")[:b * per].to(torch.int32).view(b, per)
    table = table.masked_fill(torch.arange(per, device="cuda") * page >= lengths[:, None], -1).contiguous()
    pages = b * per + 3
    state = dict(c, lengths=lengths, counts=counts, starts=starts, page_table=table, log_mass=None, rope=None,
                 positions=None, page_mass=None)
    # Token-major rows of a packed projection, seen head-major.
    packed = randn(b, nq, h + 2 * hk, d, scale=c["gain"]).to(dtype).transpose(1, 2)
    state["q"], k, v = packed.split([h, hk, hk], 1)
    if c["kind"] == "append":
        state.update(k=k, v=v, data=torch.zeros(pages, hk, page // 32, 34 * d, dtype=torch.uint8, device="cuda"))
        if c["table"]:
            angle = torch.outer(torch.arange(c["table"], device="cuda", dtype=torch.float64),
                                100.0 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2)))
            angle = torch.cat([angle, angle], 1)
            state["rope"] = (angle.sin().float(), angle.cos().float())
            if c["special"]:
                state["positions"] = (torch.arange(nq, device="cuda", dtype=torch.int32) - c["special"]).repeat(b, 1)
        if c["mass"]:
            state["log_mass"] = randint(1, 9, (b, nq)).float().log()
            state["page_mass"] = torch.zeros(pages, page, device="cuda")
        return state
    # A cache in use: every page filled by tokens of unit size.
    blocks = page // 32
    codes = [_quantised(randn(pages, hk, blocks, 32, d)) for _ in range(2)]
    state["data"] = _packed(*codes[0], *codes[1]).contiguous()
    if c["mass"]:
        state["page_mass"] = randint(1, 9, (pages, page)).float().log()
    return state


# ------------------------------------------------------------- plain form ----
def _rotated(s, x: torch.Tensor) -> torch.Tensor:
    """x cos + rot(x) sin at each token's row of the tables, in 64 bits; tokens without a row as they are."""
    x = x.double()
    if s["rope"] is None:
        return x
    sin, cos = s["rope"]
    at = s["positions"]
    if at is None:
        at = s["starts"][:, None] + torch.arange(s["nq"], device="cuda")
    held = ((at >= 0) & (at < sin.shape[0]))[:, None, :, None]
    at = at.clamp(0, sin.shape[0] - 1).long()
    low, high = x.chunk(2, -1)
    y = x * cos[at].double()[:, None] + torch.cat([-high, low], -1) * sin[at].double()[:, None]
    return torch.where(held, y, x)


def _plain_append(s) -> dict:
    b, hk, d, nq, page = (s[n] for n in ("batch", "kv_heads", "dim", "nq", "page"))
    real = torch.arange(nq, device="cuda") < s["counts"][:, None]
    keep = real[:, None, :, None]
    q = _rotated(s, s["q"]).masked_fill(~keep, 0.0).to(s["q"].dtype)
    (kc, ks), (vc, vs) = _quantised(_rotated(s, s["k"])), _quantised(s["v"].double())
    k, v = (_numbers(*t).masked_fill(~keep, 0.0).to(s["q"].dtype) for t in ((kc, ks), (vc, vs)))
    # Into the pages: a token's byte places within its block, the tokens beyond a sequence's count left out.
    at = s["starts"][:, None] + torch.arange(nq, device="cuda")
    seq, token = real.nonzero(as_tuple=True)
    at = at[seq, token].long()
    where = s["page_table"][seq, at // page].long()
    slot, base = at % 32, at % page // 32 * 34 * d
    flat = s["data"].view(-1)
    size = page // 32 * 34 * d  # of a page of one head
    row = (where * hk * size + base)[:, None, None] + torch.arange(hk, device="cuda")[:, None] * size
    pair = lambda c: (c[..., 0::2] | c[..., 1::2] << 4).transpose(1, 2)[seq, token]
    byte, part = torch.arange(d // 2, device="cuda"), torch.arange(d // 32, device="cuda")
    slot = slot[:, None, None]
    flat[row + slot * (d // 2) + byte] = pair(kc)
    flat[row + 16 * d + slot // 8 * 4 * d + byte * 8 + slot % 8] = pair(vc)
    flat[row + 32 * d + slot * (d // 32) + part] = ks.transpose(1, 2)[seq, token]
    flat[row + 33 * d + slot // 8 * (d // 4) + part * 8 + slot % 8] = vs.transpose(1, 2)[seq, token]
    out = dict(q=q, k=k, v=v)
    if s["log_mass"] is not None:
        s["page_mass"][where, at % page] = s["log_mass"][seq, token]
        out["page_mass"] = s["page_mass"]
    return out


def _plain_attend(s) -> torch.Tensor:
    b, h, hk, d, nq, page = (s[n] for n in ("batch", "heads", "kv_heads", "dim", "nq", "page"))
    # Every sequence's pages in a row, [b, hk, tokens, d].
    held = s["data"][s["page_table"].clamp(min=0)].transpose(1, 2)  # [b, hk, pages, blocks, bytes]
    kc, ks, vc, vs = _unpacked(held, d)
    k, v = (_numbers(*t).flatten(2, 4) for t in ((kc, ks), (vc, vs)))
    n = k.shape[2]
    j = torch.arange(n, device="cuda")
    i = torch.arange(nq, device="cuda")
    ok = (j < s["lengths"][:, None, None]) & (i < s["counts"][:, None])[:, :, None]
    if s["causal"]:
        ok = ok & (j <= (s["lengths"] - s["counts"])[:, None, None] + i[:, None])
    q = s["q"].float().reshape(b, hk, h // hk * nq, d)
    scores = (q @ k.transpose(-1, -2) * d ** -0.5).view(b, h, nq, n)
    if s["page_mass"] is not None:
        scores = scores + s["page_mass"][s["page_table"].clamp(min=0)].view(b, 1, 1, n)
    scores = scores.masked_fill(~ok[:, None], -math.inf)
    peak = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(peak == -math.inf, 0.0, peak))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p.view(b, hk, h // hk * nq, n) @ v
    return out.view(b, h, nq, d).to(s["q"].dtype)


# ----------------------------------------------------------------- passes ----
@functools.lru_cache(maxsize=1)
def _vgo():
    return importlib.import_module("4d_ttt_merging_amd")


@torch.no_grad()
def run(s):
    if s["kind"] == "append":
        if not own:
            return _plain_append(s)
        vgo = _vgo()
        cache = vgo.PagedCache(s["data"], s["page_mass"])
        q = vgo.cache_append(cache, s["k"], s["v"], s["page_table"], s["starts"], s["counts"], q=s["q"], rope=s["rope"],
                             positions=s["positions"], log_mass=s["log_mass"])
        k, v = vgo.cache_read(cache, s["page_table"], s["starts"], s["nq"], s["counts"], dtype=s["q"].dtype)
        out = dict(q=q, k=k, v=v)
        if s["log_mass"] is not None:
            out["page_mass"] = s["page_mass"]
        return out
    if not own:
        return _plain_attend(s)
    vgo = _vgo()
    return vgo.cached_attention(s["q"], vgo.PagedCache(s["data"], s["page_mass"]), s["page_table"], s["lengths"],
                                s["counts"], causal=s["causal"])


# ------------------------------------------------------------ work, exact ----
def work(case: dict) -> dict:
    c = {**DEFAULTS, **case}
    size = 4 if c["dtype"] == "fp32" else 2
    d, hk = c["dim"], c["kv_heads"]
    counts = c["nq"] * (0.75 if c["ragged"] and c["nq"] > 8 else 1.0)
    token = 2 * hk * 17 * d // 32  # a token's keys and values in the cache
    q = c["batch"] * counts * c["heads"] * d * size
    if c["kind"] == "append":
        tokens = c["batch"] * counts
        return {"bytes": int(2 * q + tokens * (4 * hk * d * size + 2 * token)),
                "flops": int(tokens * d * (6 * c["heads"] + 14 * hk))}
    # Lengths spread from a quarter to the whole, but never below the new tokens.
    low, high = c["nk"] / 4, float(c["nk"])
    keys = high if not c["ragged"] else max((low + high) / 2, counts)
    seen = keys - (counts - 1) / 2 if c["causal"] else keys
    return {"bytes": int(2 * q + c["batch"] * keys * token), "flops": int(4 * d * c["batch"] * c["heads"] * counts * seen)}


def _exact_numbers(x: torch.Tensor) -> torch.Tensor:
    """The cache's numbers of 64-bit values [..., dim], by the nearest of the fifteen multiples of the scale."""
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().max(-1, keepdim=True).values
    scale = torch.full_like(top, 2.0 ** -125)
    while bool((wide := (top > 7 * scale) & (scale < 2.0 ** 125)).any()):
        scale = torch.where(wide, 2 * scale, scale)
    ratio = (blocks / scale).abs().clamp(max=6.0)
    step = torch.where(ratio < 2, 0.5, torch.where(ratio < 4, 1.0, 2.0))  # (round() takes ties to the even multiple)
    return (torch.round(ratio / step) * step * blocks.sign() * scale).reshape(x.shape)


def exact(case: dict, seed: int):
    """64 bits, from the definition: rotations as complex products, one sequence and key head at a time."""
    s = prepare(case, seed)
    b, h, hk, d, nq, page = (s[n] for n in ("batch", "heads", "kv_heads", "dim", "nq", "page"))
    f64 = torch.float64
    lengths, counts = s["lengths"].tolist(), s["counts"].tolist()
    if s["kind"] == "append":
        out = dict(q=torch.zeros(b, h, nq, d, dtype=f64, device="cuda"))
        out["k"], out["v"] = (torch.zeros(b, hk, nq, d, dtype=f64, device="cuda") for _ in range(2))
        for i in range(b):
            n = counts[i]
            for name in ("q", "k"):
                x = s[name][i, :, :n].to(f64)
                if s["rope"] is not None:
                    first = 0 if s["positions"] is None else s["special"]
                    row = torch.arange(first, n, device="cuda") - first + (lengths[i] - n if s["positions"] is None else 0)
                    last = first + int((row < s["table"]).sum())
                    row = row[row < s["table"]]
                    turn = torch.complex(s["rope"][1][row, :d // 2].to(f64), s["rope"][0][row, :d // 2].to(f64))
                    turned = torch.complex(x[:, first:last, :d // 2].contiguous(), x[:, first:last, d // 2:].contiguous()) * turn
                    x[:, first:last] = torch.cat([turned.real, turned.imag], -1)
                out[name][i, :, :n] = x if name == "q" else _exact_numbers(x)
            out["v"][i, :, :n] = _exact_numbers(s["v"][i, :, :n].to(f64))
        if s["log_mass"] is not None:
            mass = s["page_mass"].to(f64)
            for i in range(b):
                for t in range(0, counts[i]):
                    place = lengths[i] - counts[i] + t
                    mass[int(s["page_table"][i, place // page]), place % page] = s["log_mass"][i, t].to(f64)
            out["page_mass"] = mass
        return out
    if h * sum(n * c for n, c in zip(lengths, counts)) > 6e9:
        return None
    levels = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=f64, device="cuda") / 2
    out = torch.zeros(b, h, nq, d, dtype=f64, device="cuda")
    for i in range(b):
        n, c = lengths[i], counts[i]
        used = s["page_table"][i, :-(-n // page)].long()
        mask = torch.arange(n, device="cuda")[None, :] <= (n - c + torch.arange(c, device="cuda"))[:, None]
        for head in range(hk):
            raw = s["data"][used, head].reshape(-1, 34 * d)
            key, value, key_scale, value_scale = raw.split([16 * d, 16 * d, d, d], 1)
            key, key_scale = key.reshape(-1, d // 2), key_scale.reshape(-1, d // 32)
            value = value.reshape(-1, 4, d // 2, 8).transpose(2, 3).reshape(-1, d // 2)
            value_scale = value_scale.reshape(-1, 4, d // 32, 8).transpose(2, 3).reshape(-1, d // 32)

            def number(code, scale):
                both = torch.empty(code.shape[0], d, dtype=f64, device="cuda")
                both[:, 0::2], both[:, 1::2] = levels[(code % 16).long()], levels[(code // 16).long()]
                return (both * torch.exp2(scale.to(f64) - 127).repeat_interleave(32, 1))[:n]
            key, value = number(key, key_scale), number(value, value_scale)
            for one in range(head * (h // hk), (head + 1) * (h // hk)):
                z = s["q"][i, one, :c].to(f64) @ key.T / math.sqrt(d)
                if s["page_mass"] is not None:
                    z = z + s["page_mass"][used].reshape(-1)[:n].to(f64)
                if s["causal"]:
                    z = torch.where(mask, z, -math.inf)
                out[i, one, :c] = torch.softmax(z, -1) @ value
    return out
