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


@pytest.mark.parametrize("dtype, d, h, hk, n, rules", [
    (BF16, 64, 64, 64, 300, dict(causal=True, cap=3.0)), (BF16, 128, 64, 8, 300, dict(docs="sorted", mass=True)),
    (F16, 64, 64, 16, 270, dict(causal=True, prefix=[90], slopes=True)), (F32, 64, 64, 64, 200, dict(buckets=16, distance=30)),
    (BF16, 64, 4, 4, 1100, dict(causal=True, buckets=32)), (BF16, 64, 2, 1, 1500, dict(mass=True, slopes=True))])
def test_gradients_of_many_tiles(vgo, device, dtype, d, h, hk, n, rules):
    """Work-groups that run over several tiles, and (few heads) work split over the other side's tiles."""
    check(vgo, *make(device, dtype, h=h, hk=hk, nq=n, nk=n, d=d, **rules))


@pytest.mark.parametrize("b, h, hk, nq, nk, d, rules", [
    (3, 8, 2, 1, 3000, 64, dict(lengths=[3000, 1, 1777], starts=[2999, 0, 1776], cap=6.0)),
    (1, 8, 8, 1, 4096, 128, dict(slopes=True)), (2, 16, 1, 4, 700, 64, dict(causal=True, buckets=32)),
    (1, 16, 1, 31, 200, 64, dict(causal=True)), (1, 16, 1, 2, 300, 64, dict(buckets=32, distance=2000)),
    (2, 4, 2, 1, 500, 64, dict(docs="mixed", mass=True)), (2, 4, 2, 7, 90, 64, dict(lengths=[0, 90]))])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_queries(vgo, device, dtype, b, h, hk, nq, nk, d, rules):
    check(vgo, *make(device, dtype, b=b, h=h, hk=hk, nq=nq, nk=nk, d=d, **rules))


def test_strides(vgo, device):
    """Packed projections, broadcast heads and batches, odd strides and offsets: the result of contiguous operands."""
    g = torch.Generator().manual_seed(1)
    packed = torch.randn(2, 90, 3, 4, 64, generator=g).bfloat16().to(device)
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
    expect = vgo.masked_attention(*(t.contiguous() for t in (q, k, v)), causal=True)
    out = vgo.masked_attention(q, k, v, causal=True)
    assert torch.equal(out, expect) and out.stride() == (90 * 256, 64, 256, 1)
    odd = [torch.randn(2, 4, 90, 67, generator=g).bfloat16().to(device)[..., 3:] for _ in range(3)]
    assert torch.equal(vgo.masked_attention(*odd), vgo.masked_attention(*(t.contiguous() for t in odd)))
    turned = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    assert torch.equal(vgo.masked_attention(*turned, causal=True), expect)
    one = [t[:1, :1].expand(2, 4, -1, -1) for t in (k, v)]
    assert torch.equal(vgo.masked_attention(q, *one), vgo.masked_attention(q, *(t.contiguous() for t in one)))
    # The gradient of what was broadcast is summed over it.
    leaf = k[:1, :1].detach().clone().requires_grad_()
    full = leaf.detach().expand(2, 4, -1, -1).clone().requires_grad_()
    grad = torch.randn(2, 4, 90, 64, generator=g).bfloat16().to(device)
    got, = torch.autograd.grad(vgo.masked_attention(q, leaf.expand(2, 4, -1, -1), v), leaf, grad)
    ref, = torch.autograd.grad(vgo.masked_attention(q, full, v), full, grad)
    assert torch.equal(got, ref.sum_to_size(leaf.shape))
    # An expanded gradient (of out.sum()).
    got, = torch.autograd.grad(vgo.masked_attention(q, full, v).sum(), full)
    ref, = torch.autograd.grad(vgo.masked_attention(q, full, v), full, torch.ones_like(grad))
    assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_masked_may_hold_anything(vgo, device, dtype):
    """NaN and infinity in padded keys, in keys and queries of no document, and in their outputs' gradients."""
    q, k, v, rules, grad = make(device, dtype, b=2, h=2, nq=150, nk=150, docs="mixed", lengths=[150, 70])
    docs = rules["key_documents"]
    rules["documents"] = docs
    dead = (docs < 0) | (torch.arange(150, device=device) >= rules["key_lengths"][:, None])
    outs = []
    for fill in (0.0, math.nan, math.inf):
        kk, vv = (t.masked_fill(dead[:, None, :, None], fill).requires_grad_() for t in (k, v))
        qq = q.masked_fill((docs < 0)[:, None, :, None], fill).requires_grad_()
        out = vgo.masked_attention(qq, kk, vv, **rules)
        g = grad.masked_fill((docs < 0)[:, None, :, None], fill)
        outs.append([out.detach(), *torch.autograd.grad(out, (qq, kk, vv), g)])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_mass_of_minus_infinity_and_the_lowest_value(vgo, device):
    q, k, v, rules, grad = make(device, BF16, nq=70, nk=140, mass=True)
    rules["log_key_mass"][::3] = -math.inf
    rules["log_key_mass"][1::3] = torch.finfo(torch.float32).min
    check(vgo, q, k, v, rules, grad)
    rules["log_key_mass"][:] = -math.inf
    assert not vgo.masked_attention(q, k, v, **rules).any()
    # A whole row at the type's lowest value is a softmax over equals.
    rules["log_key_mass"][:] = -1e30
    out = vgo.masked_attention(q, k, v, **rules)
    torch.testing.assert_close(out.float(), v.float().mean(2, keepdim=True).expand_as(out), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_no_query_no_key_no_batch(vgo, device):
    for b, nq, nk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        q, k, v, rules, grad = make(device, BF16, b=b, nq=nq, nk=nk, mass=True, slopes=True, buckets=8, distance=9)
        leaves = [t.requires_grad_() for t in (q, k, v, rules["log_key_mass"], rules["slopes"], rules["bucket_table"])]
        out = vgo.masked_attention(q, k, v, **rules)
        assert out.shape == q.shape and not out.any()
        for leaf, got in zip(leaves, torch.autograd.grad(out, leaves, grad)):
            assert got.shape == leaf.shape and not got.any()


def test_large_scores(vgo, device):
    """Logits in the hundreds, growing along the keys so that every tile moves the reference."""
    q, k, v, rules, grad = make(device, F32, nq=40, nk=300, gain=20.0)
    k = k * torch.linspace(0.1, 4.0, 300, device=device)[:, None]
    check(vgo, q, k, v, rules, grad)
    q, k, v, rules, _ = make(device, F16, nq=40, nk=300, gain=20.0)
    check(vgo, q, (k * torch.linspace(0.1, 4.0, 300, device=device)[:, None]).half(), v, rules)


def test_parameters_of_other_types(vgo, device):
    """Masses, slopes and table in the type they come in; gradients in it too."""
    q, k, v, rules, grad = make(device, BF16, h=4, nq=90, nk=90, mass=True, slopes=True, buckets=16)
    for t in (BF16, F16):
        check(vgo, q, k, v, {n: x.to(t) if isinstance(x, torch.Tensor) else x for n, x in rules.items()}, None)
        leaf = rules["bucket_table"].to(t).requires_grad_()
        out = vgo.masked_attention(q, k, v, **{**rules, "bucket_table": leaf})
        assert torch.autograd.grad(out, leaf, grad)[0].dtype == t


def test_gradient_against_differences(vgo, device):
    q, k, v, rules, grad = make(device, F32, b=1, h=2, nq=60, nk=80, causal=True, cap=3.0, mass=True, slopes=True,
                                buckets=16, distance=20, gain=2.0)
    at = dict(q=q, k=k, v=v, **{n: rules.pop(n) for n in ("log_key_mass", "slopes", "bucket_table")})
    leaves = {n: t.detach().requires_grad_() for n, t in at.items()}
    grads = dict(zip(leaves, torch.autograd.grad(vgo.masked_attention(**leaves, **rules), list(leaves.values()), grad)))
    g = torch.Generator(device=device).manual_seed(2)
    for name, t in at.items():
        direction = torch.randn(t.shape, generator=g, device=device)
        step = 2.0 ** -9
        up, down = (vgo.masked_attention(**{**at, name: t + s * direction}, **rules).double() for s in (step, -step))
        got, expect = (grads[name].double() * direction).sum(), ((up - down) / (2 * step) * grad).sum()
        # The outputs' fp32 error over the step, and the step's square.
        noise = 2e-5 * grad.abs().sum().item() / step * 2.0 ** -4
        assert abs(got - expect) <= noise, (name, got.item(), expect.item(), noise)


def test_repeats_are_the_same_bits(vgo, device):
    q, k, v, rules, grad = make(device, BF16, h=8, hk=2, nq=1000, nk=1000, causal=True, mass=True, slopes=True, buckets=32)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, rules["log_key_mass"], rules["slopes"], rules["bucket_table"])]
    rules.update(log_key_mass=leaves[3], slopes=leaves[4], bucket_table=leaves[5])
    run = lambda: torch.autograd.grad(vgo.masked_attention(*leaves[:3], **rules), leaves, grad)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_only_what_is_asked_for(vgo, device):
    """Gradients of some leaves, each what it is among all of them."""
    q, k, v, rules, grad = make(device, BF16, nq=90, nk=90, mass=True, buckets=8, distance=20)
    names = ["q", "k", "v", "log_key_mass", "bucket_table"]
    at = dict(q=q, k=k, v=v, **{n: rules.pop(n) for n in names[3:]})
    full = {n: t.detach().requires_grad_() for n, t in at.items()}
    every = dict(zip(names, torch.autograd.grad(vgo.masked_attention(**full, **rules), list(full.values()), grad)))
    for name in names:
        leaf = at[name].detach().requires_grad_()
        got, = torch.autograd.grad(vgo.masked_attention(**{**at, name: leaf}, **rules), leaf, grad)
        assert torch.equal(got, every[name]), name
    with torch.no_grad():
        assert not vgo.masked_attention(**full, **rules).requires_grad
    out = vgo.masked_attention(**full, **rules)
    with pytest.raises(RuntimeError, match="masked_attention_grad"):
        torch.autograd.grad(torch.autograd.grad(out, full["q"], grad, create_graph=True)[0].sum(), full["k"])


def test_other_stream(vgo, device):
    q, k, v, rules, grad = make(device, BF16, h=8, nq=600, nk=600, causal=True)
    expect = vgo.masked_attention(q, k, v, **rules)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [vgo.masked_attention(q, k, v, **rules) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, expect) for t in got)


def test_captured_and_replayed(vgo, device):
    """Two graphs, one of the forward and one of a training step, replayed with new inputs between eager calls."""
    q, k, v, rules, grad = make(device, BF16, b=2, h=4, hk=2, nq=300, nk=300, docs="sorted", mass=True, buckets=16)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, rules["log_key_mass"], rules["bucket_table"])]
    rules.update(log_key_mass=leaves[3], bucket_table=leaves[4])

    def step():
        out = vgo.masked_attention(*leaves[:3], **rules)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    def forward():
        with torch.no_grad():
            return vgo.masked_attention(*leaves[:3], **rules)

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        for _ in range(2):
            step(), forward()
    torch.cuda.current_stream().wait_stream(warm)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        held = step()
    with torch.cuda.graph(two):
        held_out = forward()
    for i in range(3):
        with torch.no_grad():
            for leaf in leaves:
                leaf.copy_(torch.randn(leaf.shape, device=device))
        one.replay(), two.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*held, held_out)]
        expect = step()
        assert all(torch.equal(a, b) for a, b in zip(got, [*expect, expect[0]])), i


def test_refusals(vgo, device):
    q, k, v, rules, _ = make(device, BF16, h=4, hk=2, nq=20, nk=20)
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=device)
    wrong = [
        dict(score_cap=-1.0), dict(score_cap=math.inf), dict(scale=0.0), dict(scale=math.nan), dict(prefix_lengths=i32(1)),
        dict(causal=True, prefix_lengths=i32(2)), dict(causal=True, prefix_lengths=i32(1).long()), dict(key_documents=i32(1, 20)),
        dict(documents=i32(1, 19)), dict(documents=i32(1, 20).long()), dict(key_lengths=i32(2)), dict(query_starts=i32(1, 1)),
        dict(slopes=torch.ones(3, device=device)), dict(slopes=i32(4)), dict(bucket_table=torch.ones(32, 3, device=device)),
        dict(bucket_table=torch.ones(32, device=device)), dict(bucket_table=torch.ones(31, 4, device=device)),
        dict(bucket_table=torch.ones(32, 4, device=device), max_distance=4), dict(log_key_mass=torch.ones(19, device=device)),
        dict(log_key_mass=torch.ones(20, device=device).double())]
    for more in wrong:
        with pytest.raises(ValueError):
            vgo.masked_attention(q, k, v, **more)
    for args in ((q[0], k, v), (q, k[:, :, :19], v), (q[:, :3], k, v), (q.float(), k, v), (q.double(), k.double(), v.double()),
                 (q[..., :32], k[..., :32], v[..., :32]), (q, k[:, :0], v[:, :0])):
        with pytest.raises(ValueError):
            vgo.masked_attention(*args)
    with pytest.raises(RuntimeError):
        vgo.masked_attention(q, k.cpu(), v)
    with pytest.raises(RuntimeError):
        vgo.masked_attention(q, k, v, documents=i32(1, 20).cpu())


def test_transforms(vgo, device):
    """vmap runs one call per element; forward mode and functional gradients are refused, not dropped."""
    q, k, v, rules, _ = make(device, F32, b=3, nq=20, nk=20)
    got = torch.func.vmap(lambda a, b, c: vgo.masked_attention(a[None], b[None], c[None], causal=True)[0])(q, k, v)
    assert torch.equal(got, vgo.masked_attention(q, k, v, causal=True))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: vgo.masked_attention(t, k, v).sum())(q)
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        vgo.masked_attention(forward_ad.make_dual(q, q).requires_grad_(), k, v)


def test_compiled(vgo, device):
    """Traced as one node, forward and backward."""
    q, k, v, rules, grad = make(device, F32, h=4, hk=2, nq=40, nk=40, causal=True, buckets=8, distance=12)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, rules["bucket_table"])]
    call = lambda q, k, v, t: vgo.masked_attention(q, k, v, causal=True, bucket_table=t, max_distance=12) * 2
    compiled = torch.compile(call, fullgraph=True, backend="aot_eager")
    out, ref = compiled(*leaves), call(*leaves)
    assert torch.equal(out, ref)
    for a, b in zip(torch.autograd.grad(out, leaves, grad), torch.autograd.grad(ref, leaves, grad)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [None, BF16, F16])
def test_block_under_masks(vgo, device, dtype):
    """A block's attention under attn_bias: against the same block with torch's attention on a dense bias, in inference
    and for the gradients of its parameters."""
    torch.manual_seed(0)
    block = vgo.SelfAttentionBlock(128, 2, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device)
    n = 150
    x = torch.randn(2, n, 128, device=device)
    table = torch.randn(32, 2, device=device, requires_grad=True)
    docs = (torch.arange(n, device=device) // 40).int().repeat(2, 1)
    bias = dict(causal=True, documents=docs, bucket_table=table)
    gap = torch.arange(n, device=device) - torch.arange(n, device=device)[:, None]
    ok = (gap <= 0) & (docs[0][:, None] == docs[0])

    def reference():
        wide = vgo.SelfAttentionBlock(128, 2, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device).double()
        wide.load_state_dict(block.state_dict())
        t = table.detach().double().requires_grad_()
        dense = t[oracle.bucket(gap.cpu(), 32, 128, True).to(device)].permute(2, 0, 1)
        original = torch.nn.functional.scaled_dot_product_attention
        at = torch.softmax
        import importlib
        layers = importlib.import_module("4d_ttt_merging_amd.layers")
        masked = layers.masked_attention
        layers.masked_attention = lambda q, k, v, **_: at((q @ k.transpose(-1, -2) / 8 + dense).masked_fill(~ok, -math.inf), -1) @ v
        try:
            out = wide(x.double(), attn_bias=dict())
        finally:
            layers.masked_attention = masked
        assert torch.nn.functional.scaled_dot_product_attention is original
        return out, torch.autograd.grad(out.sum(), [t, wide.attn.qkv.weight, wide.norm1.weight])

    ref, ref_grads = reference()
    with torch.autocast("cuda", dtype=dtype or BF16, enabled=dtype is not None):
        out = block(x, attn_bias=bias)
        grads = torch.autograd.grad(out.sum(), [table, block.attn.qkv.weight, block.norm1.weight])
        with torch.no_grad():
            inference = block.eval()(x, attn_bias=bias)
    # The block's products in 16 bits are off by a few steps of the type; fp32 by fp32 sums of 512.
    step = {None: 2.0 ** -16, BF16: 2.0 ** -5, F16: 2.0 ** -8}[dtype]
    for got, expect in zip((out, inference, *grads), (ref, ref, *ref_grads)):
        size = expect.abs().max()
        assert (got.double() - expect).abs().max() <= step * size
    with pytest.raises(ValueError, match="token plan"):
        block.attn(x[:1], attn_bias=bias, token_plan=object())


def test_operators_together(vgo, device):
    """A training step of a small causal model, then the same tokens one at a time over a cache: the forward with the
    dense bias added by torch, the fused bias, and the single-token form agree."""
    torch.manual_seed(0)
    b, h, hk, n, d = 2, 4, 2, 130, 64
    q, k, v, rules, grad = make(device, F32, b=b, h=h, hk=hk, nq=n, nk=n, d=d, causal=True, cap=8.0)
    table = torch.randn(32, h, device=device, requires_grad=True)
    fused = vgo.masked_attention(q, k, v, bucket_table=table, **rules)
    dense = vgo.relative_position_bias(table, n, n)
    kk, vv = (t.repeat_interleave(h // hk, 1).double() for t in (k, v))
    scores = torch.tanh(q.double() @ kk.transpose(-1, -2) / 8 / 8.0) * 8.0 + dense.double()
    future = torch.ones(n, n, device=device, dtype=torch.bool).triu(1)
    plain = torch.softmax(scores.masked_fill(future, -math.inf), -1) @ vv
    assert (fused.double() - plain).abs().max() <= 2.0 ** -17
    one, = torch.autograd.grad(fused, table, grad)
    two, = torch.autograd.grad(plain, table, grad.double())
    assert (one - two).abs().max() <= 2.0 ** -14 * two.abs().max()
    cache_k, cache_v = torch.full((b, hk, 200, d), math.nan, device=device), torch.full((b, hk, 200, d), math.nan, device=device)
    for t in range(0, n, 43):
        cache_k[:, :, :t + 1], cache_v[:, :, :t + 1] = k[:, :, :t + 1], v[:, :, :t + 1]
        length = torch.full((b,), t + 1, dtype=torch.int32, device=device)
        token = vgo.masked_attention(q[:, :, t:t + 1], cache_k, cache_v, bucket_table=table.detach(), key_lengths=length,
                                     query_starts=length - 1, **rules)
        assert (token.double() - plain[:, :, t:t + 1]).abs().max() <= 2.0 ** -17


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_slope_gradient_under_equal_rows(vgo, device, dtype, d):
    """Rows that all round their probabilities alike, where what D = dO . O is off by adds up: q = 0, slopes of 0, and
    keys told apart by their masses alone.

    Each of P, O and the dP . P that D stands for is taken with a rounding of what a rounding left out, u^2 with
    u = eps / 2, or in 32 bits; the distances weigh it.  So d slope is off by at most (2 u^2 + 2^-18) times
    T = sum over pairs of P |r| (|dO| . |v| + |dO| . sum P |v|): 2^-18 for the exponentials (2^-21 on exponents
    of at most 8), 128 products and the sums of at most 2^6 terms of 2^-24 each, T times.
    """
    n, heads = 64, 2
    mass = torch.tensor([1.0, 1.7, 3.1, 0.9, 2.3, 1.1, 5.9], dtype=torch.float64).log().float()
    nk = len(mass)
    q = torch.zeros(1, heads, n, d)
    k = torch.ones(1, heads, nk, d)
    v = torch.tensor([1.0, -1.0, 0.5, 2.0, -0.25, 0.75, 0.125])[:, None].expand(1, heads, nk, d).contiguous()
    grad = torch.zeros(1, heads, n, d)
    grad[..., 0] = 1.0
    slopes = torch.zeros(heads, device=device, requires_grad=True)
    on = lambda t: t.to(device, dtype)
    out = vgo.masked_attention(on(q), on(k), on(v), mass.to(device), slopes=slopes)
    (got,) = torch.autograd.grad(out, slopes, on(grad))

    p = torch.softmax(mass.double(), 0)
    r = (torch.arange(nk) - (nk - n + torch.arange(n))[:, None]).abs().double()
    value = v[0, 0, :, 0].double()
    expected = -(r * (p * (value - p @ value))).sum()
    terms = (r * (p * (value.abs() + p @ value.abs()))).sum()
    bound = (2 * (torch.finfo(dtype).eps / 2) ** 2 + 2.0 ** -18) * terms
    assert (got.double().cpu() - expected).abs().max() <= bound


def test_offsets_past_32_bits(vgo, device):
    """Rows of keys and values 2**23 elements apart, the last of them past 2**32, in and out of training."""
    n, apart = 600, 2 ** 23
    g = torch.Generator().manual_seed(5)
    q, k, v, grad = (torch.randn(1, 2, n, 64, generator=g).bfloat16().to(device) for _ in range(4))
    far = torch.empty(n * apart, dtype=BF16, device=device)
    held = [far.as_strided((1, 2, n, 64), (apart, 64, apart, 1), at) for at in (0, 1024)]
    for to, of in zip(held, (k, v)):
        to.copy_(of)
    results = []
    for operands in ((k, v), held):
        leaves = [t.detach().requires_grad_() for t in (q, *operands)]
        out = vgo.masked_attention(*leaves, causal=True)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, grad)])
        with torch.no_grad():
            results[-1].append(vgo.masked_attention(q[:, :, -1:], *operands))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_lengths_and_positions_out_of_range(vgo, device):
    """Lengths, prefixes and positions past the keys, or negative, are what they are clamped to."""
    most, least = 2 ** 31 - 1, -2 ** 31
    q, k, v, _, _ = make(device, BF16, b=2, nq=70, nk=130)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    run = lambda **rules: vgo.masked_attention(q, k, v, **rules)
    assert torch.equal(run(key_lengths=i32(most, least)), run(key_lengths=i32(130, 0)))
    assert torch.equal(run(causal=True, prefix_lengths=i32(most, least)), run(causal=True, prefix_lengths=i32(130, 0)))
    assert torch.equal(run(causal=True, query_starts=i32(most, least)), run(causal=True, query_starts=i32(130, -70)))
    table = torch.randn(32, 2, device=device)
    far = run(bucket_table=table, slopes=torch.zeros(2, device=device), query_starts=i32(most, least))
    assert torch.equal(far, run(bucket_table=table, slopes=torch.zeros(2, device=device), query_starts=i32(10 ** 6, -10 ** 6)))


def test_two_streams_at_once(vgo, device):
    """Calls in flight together, each split over the keys with partial states of its own."""
    q, k, v, rules, grad = make(device, BF16, b=1, h=4, nq=500, nk=2000, causal=True, slopes=True)

    def step(scale):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = vgo.masked_attention(*leaves, **{**rules, "scale": scale})
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    expect = [step(0.125), step(0.25)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step((0.125, 0.25)[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, expect[i]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_padded_batch_in_training(vgo, device, dtype):
    """Sequences of 0, 1, 64 and 100 of 100 keys: each alone, and what lies behind its keys without gradient."""
    lengths = [0, 1, 64, 100]
    q, k, v, _, grad = make(device, dtype, b=4, nq=100, nk=100, seed=3)
    k, v = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        k[b, :, n:], v[b, :, n:] = math.nan, math.nan
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = vgo.masked_attention(*leaves, key_lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    grads = torch.autograd.grad(out, leaves, grad)
    assert not out[0].any() and not any(g[0].any() for g in grads)
    for b, n in enumerate(lengths[1:], 1):
        assert not grads[1][b, :, n:].any() and not grads[2][b, :, n:].any()
        start = torch.tensor([0], dtype=torch.int32, device=device)
        res, bound = oracle.attention(q[b:b + 1], k[b:b + 1, :, :n], v[b:b + 1, :, :n], grad=grad[b:b + 1], query_starts=start)
        for name, got in zip(("out", "q", "k", "v"), (out.detach(), *grads)):
            got = got[b:b + 1] if name in ("out", "q") else got[b:b + 1, :, :n]
            within(got, res[name], bound[name], f"{name} of {n} keys")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("reach", [0.05, 0.27, 0.29, 0.74, 0.76, 3.0])
def test_scores_around_the_caps_series(vgo, device, dtype, reach):
    """Caps that put the largest score on either side of where the tanh is taken another way."""
    q, k, v, rules, grad = make(device, dtype, nq=70, nk=130, causal=True)
    largest = (q.double() @ k.double().transpose(-1, -2) / 8).abs().max().item()
    check(vgo, q, k, v, {**rules, "score_cap": largest / reach}, grad)
