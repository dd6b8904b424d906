"""Masked attention and its gradients against the 64-bit oracle, within its elementwise bounds."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import masked_attention as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(device, dtype, b=1, h=2, hk=2, nq=65, nk=129, d=64, seed=0, gain=1.0, mass=False, slopes=False, buckets=0,
         both=True, distance=128, causal=False, prefix=None, docs=None, lengths=None, starts=None, cap=None, scale=None):
    """(q, k, v, keyword arguments, gradient of the output), on the device."""
    g = torch.Generator().manual_seed(seed)
    draw = lambda *shape: torch.randn(*shape, generator=g)
    q = (draw(b, nq, h, d) * gain).to(dtype).transpose(1, 2)
    k, v, = (draw(b, nk, hk, d).to(dtype).transpose(1, 2) for _ in range(2))
    grad = draw(b, nq, h, d).to(dtype).transpose(1, 2)
    rules = dict(causal=causal, score_cap=cap, scale=scale)
    if mass:
        rules["log_key_mass"] = torch.randint(1, 9, (nk,), generator=g).float().log()
    if slopes:
        rules["slopes"] = 2.0 ** -torch.arange(1.0, h + 1)
    if buckets:
        rules.update(bucket_table=draw(buckets, h), bidirectional=both, max_distance=distance)
    int32 = lambda t: torch.tensor(t, dtype=torch.int32)
    if prefix is not None:
        rules["prefix_lengths"] = int32(prefix)
    if docs == "sorted":
        kd = (torch.rand(b, nk, generator=g) < 0.06).cumsum(1).int()
        rules.update(documents=kd[:, -nq:].contiguous() if nq <= nk else torch.cat([kd, kd[:, :nq - nk]], 1),
                     key_documents=kd)
    elif docs == "mixed":  # in any order, some of nobody
        rules.update(documents=torch.randint(-1, 4, (b, nq), generator=g).int(),
                     key_documents=torch.randint(-1, 4, (b, nk), generator=g).int())
    if lengths is not None:
        rules["key_lengths"] = int32(lengths)
    if starts is not None:
        rules["query_starts"] = int32(starts)
    rules = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in rules.items()}
    return q.to(device), k.to(device), v.to(device), rules, grad.to(device)


def within(got, expected, bound, what):
    got = got.double().cpu()
    assert got.shape == expected.shape
    assert torch.isfinite(got).all(), what
    off = (got - expected).abs()
    # Both sides of an exact zero are zero; the smallest normal of the 16-bit types for what rounds to less.
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 1e-7, f"{what}: off by {worst:.3e} beyond its bound, {off.max():.3e} in all"


def check(vgo, q, k, v, rules, grad=None):
    leaves = {}
    if grad is not None:
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        leaves = dict(q=q, k=k, v=v)
        rules = dict(rules)
        for n in ("log_key_mass", "slopes", "bucket_table"):
            if rules.get(n) is not None:
                rules[n] = leaves[n] = rules[n].detach().requires_grad_()
    out = vgo.masked_attention(q, k, v, **rules)
    assert out.dtype == q.dtype and out.shape == q.shape
    res, bound = oracle.attention(q, k, v, grad=grad, **rules)
    within(out.detach(), res["out"], bound["out"], "out")
    if grad is not None:
        for name, got in zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)):
            assert got.dtype == leaves[name].dtype
            within(got, res[name], bound[name], f"gradient of {name}")
    return out


SIZES = [(1, 1), (1, 64), (1, 200), (3, 5), (31, 65), (32, 32), (33, 64), (64, 63), (65, 129), (130, 70), (300, 333)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq, nk", SIZES)
def test_sizes(vgo, device, dtype, d, nq, nk):
    check(vgo, *make(device, dtype, b=2, h=4, hk=2, nq=nq, nk=nk, d=d, seed=nq + nk)[:4])


RULES = {
    "causal": dict(causal=True),
    "causal_more_queries": dict(causal=True, nq=200, nk=129),
    "prefix": dict(causal=True, prefix=[40, 129], b=2, nq=129),
    "prefix_of_zero_and_over": dict(causal=True, prefix=[0, 1000], b=2, nq=129),
    "documents": dict(docs="sorted", nq=200, nk=200),
    "documents_mixed": dict(docs="mixed", b=2, nq=150, nk=140),
    "causal_documents": dict(docs="sorted", nq=200, nk=200, causal=True, prefix=[30]),
    "lengths": dict(lengths=[0, 1, 100], starts=[0, 0, 35], b=3),
    "lengths_causal": dict(lengths=[64, 129], starts=[-30, 64], b=2, causal=True),
    "cap": dict(cap=4.0, gain=4.0),
    "cap_small_scores": dict(cap=50.0, scale=0.01),
    "mass": dict(mass=True),
    "slopes": dict(slopes=True, h=4),
    "buckets": dict(buckets=32, distance=40, nq=200, nk=200),
    "buckets_far": dict(buckets=16, distance=16, nq=40, nk=400),
    "buckets_behind": dict(buckets=32, both=False, distance=100, nq=160, nk=200, causal=True),
    "buckets_starts": dict(buckets=8, distance=300, b=2, starts=[-250, 400]),
    "everything": dict(b=2, h=4, hk=2, nq=150, nk=180, causal=True, prefix=[20, 90], docs="sorted", lengths=[180, 131],
                       cap=5.0, gain=2.0, mass=True, slopes=True, buckets=32, distance=64, scale=0.2),
}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rule", list(RULES))
def test_rules(vgo, device, dtype, rule):
    check(vgo, *make(device, dtype, **RULES[rule])[:4])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq, nk", [(1, 1), (5, 3), (64, 64), (130, 70), (70, 261)])
def test_gradients_of_sizes(vgo, device, dtype, d, nq, nk):
    check(vgo, *make(device, dtype, b=2, h=4, hk=2, nq=nq, nk=nk, d=d, seed=nq + nk))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rule", list(RULES))
def test_gradients_of_rules(vgo, device, dtype, rule):
    check(vgo, *make(device, dtype, **RULES[rule]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_everything_at_once_wide(vgo, device, dtype, d):
    check(vgo, *make(device, dtype, d=d, **RULES["everything"]))


# Many heads: work-groups of four waves, with 32 (128 channels, fp32) or, from 256 queries a head on, 64 queries each.
@pytest.mark.parametrize("dtype, d, h, nq, rules", [
    (BF16, 64, 256, 130, dict(causal=True)), (F16, 64, 256, 300, dict(causal=True, cap=3.0)),
    (BF16, 64, 256, 257, dict(docs="mixed", buckets=8, distance=30)), (BF16, 128, 256, 150, dict(docs="sorted", slopes=False)),
    (BF16, 128, 128, 290, dict(causal=True, prefix=[100], mass=True)), (F32, 64, 256, 129, dict(causal=True)),
    (F32, 128, 256, 140, dict(docs="sorted", mass=True))])
def test_many_heads(vgo, device, dtype, d, h, nq, rules):
    check(vgo, *make(device, dtype, h=h, hk=h // 4, nq=nq, nk=200, d=d, **rules)[:4])
