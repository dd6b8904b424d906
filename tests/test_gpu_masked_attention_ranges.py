"""Masked attention at the ends of its ranges: masses that keep keys out, caps, positions, lengths and sizes."""
from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import masked_attention as oracle
from tests.test_gpu_masked_attention import BF16, F16, F32, make, within

pytestmark = pytest.mark.gpu


def check(vgo, q, k, v, rules, grad=None):
    """Against the oracle, within its bounds.  They count a half step relative to a value: score gradients are held
    in the operands' type for dQ and dK, and those of f16 below 2^-14 are off by up to 2^-25 each, whatever their size."""
    leaves = {}
    if grad is not None:
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        leaves, rules = dict(q=q, k=k, v=v), dict(rules)
        for n in ("log_key_mass", "slopes", "bucket_table"):
            if rules.get(n) is not None:
                rules[n] = leaves[n] = rules[n].detach().requires_grad_()
    out = vgo.masked_attention(q, k, v, **rules)
    res, bound = oracle.attention(q, k, v, grad=grad, **rules)
    within(out.detach(), res["out"], bound["out"], "out")
    if grad is None:
        return
    if q.dtype == F16:
        b, h, nq, d = q.shape
        step = 2.0 ** -25 * (rules.get("scale") or d ** -0.5)
        q64, k64 = (t.detach().double().cpu().abs() for t in (q, k))
        group = h // k.shape[1]
        bound["q"] = bound["q"] + step * k64.sum(2, keepdim=True).repeat_interleave(group, 1)
        bound["k"] = bound["k"] + step * q64.reshape(b, k.shape[1], group * nq, d).sum(2, keepdim=True)
    for name, got in zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)):
        within(got, res[name], bound[name], f"gradient of {name}")


def equal_keys(q, k, v, grad, seen):
    """(results, bounds) of attention whose keys' scores are all equal: the mean over the keys that a row sees
    ([nq, nk]), one key head a head, scale 1 / sqrt(d).

    P is 1 / n up to the exponential, the logarithm and a division of the hardware's, 2^-22 each: 2^-20 with what
    they multiply.  Sums of n, d and the rows' terms lose half a step of fp32 a term; P, score gradients and results
    of 16 bits half a step of the type each."""
    u, u32 = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    rounded = 0.0 if q.dtype == F32 else u
    q, k, v, grad = (t.detach().double().cpu() for t in (q, k, v, grad))
    d, nq, nk = q.shape[-1], q.shape[2], k.shape[2]
    p = seen.double() / seen.sum(1, keepdim=True).clamp(min=1)
    kappa = 2.0 ** -20 + (nk + nq + 2 * d) * u32
    out = p @ v
    dp, delta = grad @ v.transpose(-1, -2), (grad * out).sum(-1, keepdim=True)
    dz = p * (dp - delta)
    res = dict(out=out, q=dz @ k * d ** -0.5, k=dz.transpose(-1, -2) @ q * d ** -0.5, v=p.T @ grad,
               log_key_mass=dz.sum((0, 1, 2)))
    a = p @ v.abs()
    e_out = (rounded + kappa) * a + u * out.abs()
    size = grad.abs() @ v.abs().transpose(-1, -2) + (grad.abs() * a).sum(-1, keepdim=True)
    # D comes from the output as rounded (and, in 16 bits, from what that took, so this is more than it loses).
    e_dz = p * ((grad.abs() * e_out).sum(-1, keepdim=True) + kappa * size)
    e_ds = e_dz + (rounded + kappa) * dz.abs()
    bound = dict(out=e_out, q=e_ds @ k.abs() * d ** -0.5 + u * res["q"].abs(),
                 k=e_ds.transpose(-1, -2) @ q.abs() * d ** -0.5 + u * res["k"].abs(),
                 v=(rounded + kappa) * (p.T @ grad.abs()) + u * res["v"].abs(),
                 log_key_mass=(e_dz + kappa * dz.abs()).sum((0, 1, 2)))
    return res, bound


def check_equal_keys(vgo, q, k, v, grad, mass, causal):
    nq, nk = q.shape[2], k.shape[2]
    seen = torch.arange(nk) <= nk - nq + torch.arange(nq)[:, None] if causal else torch.ones(nq, nk, dtype=torch.bool)
    res, bound = equal_keys(q, k, v, grad, seen)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, mass)]
    out = vgo.masked_attention(*leaves, causal=causal)
    within(out.detach(), res["out"], bound["out"], "out")
    for name, got in zip(("q", "k", "v", "log_key_mass"), torch.autograd.grad(out, leaves, grad)):
        within(got, res[name], bound[name] + torch.finfo(got.dtype).eps / 2 * res[name].abs(), f"gradient of {name}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("offset", [-1e5, -1e6, -1e9, 1e7])
@pytest.mark.parametrize("nq, nk, causal", [(70, 140, False), (300, 300, True), (5, 1000, False)])
def test_gradients_under_a_common_mass(vgo, device, dtype, offset, nq, nk, causal):
    """Every key's mass the same large number: the row's statistics hold the logarithm of its few terms beside it."""
    q, k, v, _, grad = make(device, dtype, nq=nq, nk=nk)
    check_equal_keys(vgo, torch.zeros_like(q), k, v, grad, torch.full((nk,), offset, device=device), causal)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_whose_masses_are_all_the_lowest_value(vgo, device, dtype, kind, causal):
    """torch.finfo(t).min is a number: where every key of a row has it, scores vanish beside it and the row is a mean."""
    q, k, v, _, grad = make(device, dtype, nq=70, nk=140)
    check_equal_keys(vgo, q, k, v, grad, torch.full((140,), torch.finfo(kind).min, dtype=kind, device=device), causal)


def test_lowest_masses_before_others(vgo, device):
    """Left padding by the lowest value under a causal mask: rows of the padding take its mean, the others none of it."""
    q, k, v, _, grad = make(device, F32, nq=140, nk=140)
    mass = torch.zeros(140, device=device)
    mass[:75] = torch.finfo(F32).min
    out = vgo.masked_attention(q, k, v, mass, causal=True)
    seen = torch.arange(75) <= torch.arange(75)[:, None]
    res, bound = equal_keys(q[:, :, :75], k[:, :, :75], v[:, :, :75], grad[:, :, :75], seen)
    within(out[:, :, :75], res["out"], bound["out"], "out of the padding")
    res, bound = oracle.attention(q[:, :, 75:], k[:, :, 75:], v[:, :, 75:], causal=True)
    within(out[:, :, 75:], res["out"], bound["out"], "out behind the padding")


def test_lowest_values_of_a_table_and_masses(vgo, device):
    """A table whose every bucket is the type's lowest value, alone and beside such masses: means too."""
    q, k, v, _, grad = make(device, BF16, nq=70, nk=140)
    res, bound = equal_keys(q, k, v, grad, torch.ones(70, 140, dtype=torch.bool))
    table = torch.full((32, 2), torch.finfo(F32).min, device=device)
    for mass in (None, torch.full((140,), torch.finfo(BF16).min, dtype=BF16, device=device)):
        within(vgo.masked_attention(q, k, v, mass, bucket_table=table), res["out"], bound["out"], "out")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [120.0, 200.0, 1e4, 1e6, 1e8, 1e20, 1e30, 3e38])
def test_caps_far_above_the_scores(vgo, device, dtype, d, cap):
    """A cap that no score comes near leaves the scores as they are."""
    q, k, v, rules, grad = make(device, dtype, nq=70, nk=130, d=d, causal=True, gain=3.0)
    check(vgo, q, k, v, {**rules, "score_cap": cap}, grad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gain", [30.0, 300.0])
def test_large_scores_under_large_caps(vgo, device, dtype, gain):
    """Scores of hundreds, some past 0.3 of a cap of 1,000."""
    q, k, v, rules, grad = make(device, dtype, nq=70, nk=130, gain=gain)
    check(vgo, q, k, v, {**rules, "score_cap": 1000.0}, grad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", [1e-3, 1e-10, 1e-30, 1e-44, 1e-60])
def test_caps_far_below_the_scores(vgo, device, dtype, cap):
    """Scores cut to next to nothing: all keys alike, and no gradient through a tanh that is flat."""
    q, k, v, rules, grad = make(device, dtype, nq=70, nk=130)
    check(vgo, q, k, v, {**rules, "score_cap": cap}, grad)


@pytest.mark.parametrize("n", [70, 5000, 70000])
def test_many_improbable_keys_in_half_precision(vgo, device, n):
    """One key with all but 22.5 * 2^-24 of the weight for each of the others, and a value of 0: the output is the
    others' alone, whose weights have all their bits where the largest leaves them above f16's smallest normal number."""
    q, k, v, _, _ = make(device, F16, h=1, hk=1, nq=40, nk=n)
    v = v + 2.0
    v[:, :, 0] = 0.0
    mass = torch.full((n,), math.log(22.5) - 24.0 * math.log(2.0), device=device)
    mass[0] = 0.0
    q = torch.zeros_like(q)
    out = vgo.masked_attention(q, k, v, mass)
    res, bound = oracle.attention(q, k, v, mass)
    # (Scaled, so that small outputs count beside within()'s 1e-7; half a step of f16's subnormals is 2^-25.)
    within(out.double() * 2.0 ** 20, res["out"] * 2.0 ** 20, (bound["out"] + 2.0 ** -25) * 2.0 ** 20, "out")


@pytest.mark.parametrize("gain", [30.0, 300.0])
def test_large_scores_in_half_precision(vgo, device, gain):
    q, k, v, rules, grad = make(device, F16, nq=70, nk=130, gain=gain)
    check(vgo, q, k, v, {**rules, "score_cap": 1000.0}, grad)
    check(vgo, q, k, v, rules, grad)


RULES_F16 = ["causal", "causal_more_queries", "prefix", "documents", "documents_mixed", "causal_documents", "lengths",
             "lengths_causal", "cap", "cap_small_scores", "mass", "slopes", "buckets", "buckets_far", "buckets_behind",
             "buckets_starts", "everything"]


@pytest.mark.parametrize("rule", RULES_F16)
def test_rules_and_gradients_in_half_precision(vgo, device, rule):
    from tests.test_gpu_masked_attention import RULES
    check(vgo, *make(device, F16, **RULES[rule]))


@pytest.mark.parametrize("b, h, hk, nq, nk, d, rules", [
    (3, 8, 2, 1, 3000, 64, dict(lengths=[3000, 1, 1777], starts=[2999, 0, 1776], cap=6.0)),
    (1, 8, 8, 1, 4096, 128, dict(slopes=True)), (2, 16, 1, 4, 700, 64, dict(causal=True, buckets=32)),
    (2, 4, 2, 1, 500, 64, dict(docs="mixed", mass=True)), (2, 4, 2, 7, 90, 64, dict(lengths=[0, 90]))])
def test_few_queries_in_half_precision(vgo, device, b, h, hk, nq, nk, d, rules):
    check(vgo, *make(device, F16, b=b, h=h, hk=hk, nq=nq, nk=nk, d=d, **rules))


@pytest.mark.parametrize("h, hk, buckets, both, distance", [
    (8, 1, 64, True, 500), (8, 1, 32, False, 512), (16, 1, 16, True, 500), (4, 1, 64, False, 1000), (16, 1, 32, True, 128),
    (18, 1, 32, True, 128), (32, 1, 8, True, 40)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_queries_with_tables_that_fill_the_lds(vgo, device, dtype, h, hk, buckets, both, distance):
    """128 channels, where the heads of a group, packed into a task, would bring more tables than beside the tiles fit."""
    check(vgo, *make(device, dtype, h=h, hk=hk, nq=1, nk=300, d=128, buckets=buckets, both=both, distance=distance))


def test_documents_of_no_token(vgo, device):
    """Document masks beside no queries, no keys or no batch."""
    for b, nq, nk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        q, k, v, rules, grad = make(device, BF16, b=b, nq=nq, nk=nk, docs="mixed", mass=True, slopes=True, buckets=8, distance=9)
        leaves = [t.requires_grad_() for t in (q, k, v, rules["log_key_mass"], rules["slopes"], rules["bucket_table"])]
        out = vgo.masked_attention(q, k, v, **rules)
        assert out.shape == q.shape and not out.any()
        for leaf, got in zip(leaves, torch.autograd.grad(out, leaves, grad)):
            assert got.shape == leaf.shape and not got.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq", [1, 40, 100])
@pytest.mark.parametrize("start, at", [(10 ** 6, 129), (-10 ** 6, 0), (2 ** 31 - 1, 129), (-2 ** 31, 0)])
def test_slopes_at_positions_far_from_the_keys(vgo, device, dtype, nq, start, at):
    """A position beyond the keys differs from that of the nearest one by what a softmax leaves out: all of its rows
    attend as from there, and the slopes' gradient, whose score gradients add up to nothing in a row, is the same."""
    q, k, v, rules, grad = make(device, dtype, nq=nq, nk=130, slopes=True)
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=device)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, rules["slopes"])]
    out = vgo.masked_attention(*leaves[:3], slopes=leaves[3], query_starts=i32(start))
    grads = torch.autograd.grad(out, leaves, grad)
    total, bounds = {}, {}
    for i in range(nq):
        res, bound = oracle.attention(q[:, :, i:i + 1], k, v, slopes=rules["slopes"], query_starts=i32(at),
                                      grad=grad[:, :, i:i + 1])
        within(out.detach()[:, :, i:i + 1], res["out"], bound["out"], f"out of row {i}")
        within(grads[0][:, :, i:i + 1], res["q"], bound["q"], f"gradient of q, row {i}")
        for n in ("k", "v", "slopes"):
            total[n], bounds[n] = total.get(n, 0.0) + res[n], bounds.get(n, 0.0) + bound[n]
    for n, got in zip(("k", "v", "slopes"), grads[1:]):
        within(got, total[n], bounds[n] + torch.finfo(got.dtype).eps / 2 * total[n].abs(), f"gradient of {n}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("start", [-40, -3, 60, 128, 200])
def test_slopes_of_rows_on_both_sides_of_the_keys_ends(vgo, device, dtype, d, start):
    check(vgo, *make(device, dtype, b=2, nq=100, nk=130, d=d, slopes=True, starts=[start, 10], lengths=[130, 70]))


def uniform_parameters(heads=2, n=256, d=64):
    """q = 0 and no other rule: P = 1 / 256, values of whole numbers whose mean is one, gradients of whole numbers, so that
    every dZ is a whole multiple of 2^-8 and their sums are exact in fp32."""
    g = torch.Generator().manual_seed(11)
    q = torch.zeros(1, heads, n, d)
    k = torch.randn(1, heads, n, d, generator=g)
    v = torch.randint(-4, 5, (1, heads, n // 2, d), generator=g).float()
    v = torch.cat([v, 2.0 - v], 2)[:, :, torch.randperm(n, generator=g)]  # a mean of 1
    grad = torch.randint(-2, 3, (1, heads, n, d), generator=g).float()
    return q, k, v, grad


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_parameter_gradients_that_are_exact(vgo, device, dtype):
    """Gradients of masses, slopes and table where every term is exact but for P's exponential, the same in all rows:
    2^-20 of the result, and 2^-22 of the terms for what fp32 sums may lose.  A term is 2^-22 of all terms and more, many
    times that on average: one left out or counted twice shows."""
    q, k, v, grad = uniform_parameters()
    n, heads, buckets = 256, 2, 32
    on = lambda t: t.to(device, dtype)
    mass, slopes, table = (torch.zeros(*s, device=device, requires_grad=True) for s in ((n,), (heads,), (buckets, heads)))
    dp = (grad.double() @ v.double().transpose(-1, -2))[0]
    dz = (dp - grad.double()[0].sum(-1, keepdim=True)) / n
    gap = torch.arange(n) - torch.arange(n)[:, None]
    which = oracle.bucket(gap, buckets, 128, True)
    expected = [dz.sum((0, 1)), -(dz * gap.abs()).sum((1, 2)),
                torch.stack([(dz * (which == t)).sum((1, 2)) for t in range(buckets)])]
    terms = {"masses": dz.abs().sum((0, 1)), "masses alone": dz.abs().sum((0, 1)), "slopes": (dz * gap).abs().sum((1, 2)),
             "table": torch.stack([(dz * (which == t)).abs().sum((1, 2)) for t in range(buckets)])}
    # Slopes and tables together, and masses alone: other kernels.
    out = vgo.masked_attention(on(q), on(k), on(v), mass, slopes=slopes, bucket_table=table)
    got = torch.autograd.grad(out, (mass, slopes, table), on(grad))
    alone = torch.autograd.grad(vgo.masked_attention(on(q), on(k), on(v), mass), mass, on(grad))
    for name, a, b in zip(("masses", "slopes", "table", "masses alone"), (*got, *alone), (*expected, expected[0])):
        off = (a.double().cpu() - b).abs()
        assert (off <= 2.0 ** -20 * b.abs() + 2.0 ** -22 * terms[name]).all(), (name, off.max().item())
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rules", [{}, dict(docs="sorted", mass=True), dict(causal=True, prefix=[4500], cap=8.0)])
def test_more_than_64_tiles_a_task(vgo, device, dtype, rules):
    """2,048 single rows over 4,500 keys that they share by strides: a task to a row and 71 tiles a task, unsplit."""
    q, k, v, more, _ = make(device, dtype, h=1, nq=1, nk=4500, hk=1, **rules)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(1, 2048, 1, 64, generator=g).to(device, dtype)
    out = vgo.masked_attention(q, k.expand(-1, 2048, -1, -1), v.expand(-1, 2048, -1, -1), **more)
    some = torch.arange(0, 2048, 37)
    res, bound = oracle.attention(q[:, some], k.expand(-1, len(some), -1, -1), v.expand(-1, len(some), -1, -1), **more)
    within(out[:, some], res["out"], bound["out"], "out")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("h, nq, nk, rules", [(2100, 1, 70, dict(slopes=False)), (300, 30, 100, dict(docs="mixed")),
                                              (64, 130, 4300, dict(causal=True)), (16, 40, 9000, dict(mass=True))])
def test_gradients_of_one_key_head(vgo, device, dtype, h, nq, nk, rules):
    """Many heads on one key head, few of them or long keys: units and tiles past 64 a split, and splits past a few."""
    check(vgo, *make(device, dtype, h=h, hk=1, nq=nq, nk=nk, **rules))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_large_equal_scores(vgo, device, dtype, causal):
    """Scores of 2^15, all the same, without a bias; and masses of 1e6 under slopes and a table of zeros."""
    q, k, v, _, grad = make(device, dtype, nq=150, nk=150)
    seen = torch.arange(150) <= torch.arange(150)[:, None] if causal else torch.ones(150, 150, dtype=torch.bool)
    same = [torch.full_like(t, 64.0).requires_grad_() for t in (q, k)]
    v = v.detach().requires_grad_()
    res, bound = equal_keys(*same, v, grad, seen)
    out = vgo.masked_attention(*same, v, causal=causal)
    within(out.detach(), res["out"], bound["out"], "out")
    for name, got in zip(("q", "k", "v"), torch.autograd.grad(out, (*same, v), grad)):
        within(got, res[name], bound[name], f"gradient of {name}")
    zeros = lambda *shape: torch.zeros(*shape, device=device, requires_grad=True)
    leaves = [torch.zeros_like(q).requires_grad_(), k.requires_grad_(), v, torch.full((150,), 1e6, device=device).requires_grad_()]
    res, bound = equal_keys(*leaves[:3], grad, seen)
    for more in (dict(slopes=zeros(2)), dict(slopes=zeros(2), bucket_table=zeros(32, 2))):
        out = vgo.masked_attention(*leaves[:3], leaves[3], causal=causal, **more)
        within(out.detach(), res["out"], bound["out"], "out")
        grads = torch.autograd.grad(out, [*leaves, *more.values()], grad)
        for name, got in zip(("q", "k", "v", "log_key_mass"), grads):
            within(got, res[name], bound[name] + torch.finfo(got.dtype).eps / 2 * res[name].abs(), f"gradient of {name}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rules", [{}, dict(causal=True, mass=True), dict(docs="mixed", cap=5.0), dict(nq=3, nk=300)])
def test_buckets_that_keep_pairs_apart(vgo, device, dtype, rules):
    """Entries of -inf in the table: a mask by distance, which leaves some rows nothing, without gradient for them."""
    q, k, v, more, grad = make(device, dtype, **{**dict(nq=150, nk=150, buckets=16, distance=60), **rules})
    more["bucket_table"][8:] = -math.inf   # the keys ahead,
    more["bucket_table"][0] = -math.inf    # the query's own
    more["bucket_table"][3:6, 1] = -math.inf  # and, of one head, some behind
    check(vgo, q, k, v, more, grad)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masses_of_keys_that_nothing_reads(vgo, device, dtype):
    """NaN and infinities in the masses of padded keys."""
    q, k, v, rules, grad = make(device, dtype, b=2, nq=100, nk=150, lengths=[150, 120], mass=True, docs="mixed")
    rules["key_lengths"] = rules["key_lengths"].clamp(max=120)
    mass = rules.pop("log_key_mass")
    results = []
    for fill in (0.0, math.nan, math.inf):
        leaf = torch.cat([mass[:120], torch.full_like(mass[120:], fill)]).requires_grad_()
        leaves = [t.detach().requires_grad_() for t in (q, k, v)] + [leaf]
        out = vgo.masked_attention(*leaves, **rules)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, grad)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def drawn(seed):
    """Keyword arguments of make() with rules, sizes and positions drawn together."""
    r = random.Random(seed)
    size = lambda most: int(round(math.exp(r.uniform(0.0, math.log(most)))))
    hk, b = r.choice([1, 2, 3]), r.choice([1, 1, 2, 3])
    nq = r.choice([1, 2, size(31), size(400)])
    nk = r.choice([size(700), nq])
    case = dict(b=b, h=hk * r.choice([1, 1, 2, 4, 5]), hk=hk, nq=nq, nk=nk, d=r.choice([64, 128]), seed=seed,
                gain=r.choice([0.5, 1.0, 2.0, 6.0]), causal=r.random() < 0.5, mass=r.random() < 0.4, slopes=r.random() < 0.4,
                cap=r.choice([None, None, 0.5, 3.0, 50.0, 300.0]), scale=r.choice([None, None, 0.05, 0.3]))
    if case["causal"] and r.random() < 0.4:
        case["prefix"] = [r.randint(-3, nk + 5) for _ in range(b)]
    if r.random() < 0.4:
        case["docs"] = "mixed" if nq > 2 * nk else r.choice(["mixed", "sorted"])
    if r.random() < 0.4:
        case["lengths"] = [r.choice([0, nk, r.randint(0, nk + 3)]) for _ in range(b)]
    if r.random() < 0.4:
        case["starts"] = [r.randint(-nq - 5, nk + 5) for _ in range(b)]
    if r.random() < 0.4:
        both = r.random() < 0.6
        buckets = r.choice([8, 16, 32, 64] if both else [2, 7, 16, 33, 64])
        alone = buckets // 2 // 2 if both else buckets // 2
        case.update(buckets=buckets, both=both, distance=r.choice([alone + r.randint(1, 20), alone + 128, 300]))
    return case


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("seed", range(40))
def test_drawn_rules(vgo, device, dtype, seed):
    check(vgo, *make(device, dtype, **drawn(seed)))
