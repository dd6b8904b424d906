"""Blocks that stream through a paged cache, and the cache's operators in a user's surroundings: autocast, streams, graphs,
devices, tracing, autograd."""
from __future__ import annotations

import pytest
import torch

from oracle import paged_cache as oracle
from tests.conftest import import_package

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("dtype", [None, BF16, F16])
@pytest.mark.parametrize("heads", [2, 1])
@pytest.mark.parametrize("prefix_tokens", [0, 5])
def test_a_block_streams_frames(vgo, device, dtype, heads, prefix_tokens):
    """Three frames of a scene, one after the other, then one token: against the block's steps in 64 bits over the numbers
    that the cache holds (`cache_read`), which are the nearest to the block's own keys."""
    layers = import_package("layers")
    torch.manual_seed(0)
    dim, (h, w) = 128, (6, 7)
    d, n = dim // heads, prefix_tokens + 42
    block = vgo.SelfAttentionBlock(dim, heads, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device).eval()
    wide = vgo.SelfAttentionBlock(dim, heads, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device).eval()
    wide.load_state_dict(block.state_dict())
    wide = wide.double()
    sin, cos = layers.rope_sincos(h, w, d, device=device)
    cache = vgo.PagedCache.empty(16, heads, d, page_size=32, device=device)
    table = int32([[3, 1, 8, 11, 0], [2, 9, 4, 5, 10]], device)
    # The masked blocks' bound: under autocast LayerNorm's output, the projections, q, the probabilities, the attended
    # values and the MLP's hidden layer are rounded in turn, about 16 half steps; fp32's products of 128 to 512 terms 2^-16.
    step = {None: 2.0 ** -16, BF16: 2.0 ** -4, F16: 2.0 ** -7}[dtype]
    steps = [(n, None), (n, None), (n, [n, 20]), (1, None)]
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    for count, counts in steps:
        x = torch.randn(2, count, dim, device=device)
        rope, positions = ((sin, cos), None) if count > 1 else ((sin, cos), int32([[7], [-1]], device))
        given = None if counts is None else int32(counts, device)
        lengths = lengths + (count if given is None else given)
        with torch.no_grad(), torch.autocast("cuda", dtype=dtype or BF16, enabled=dtype is not None):
            out = block(x, rope, cached=dict(cache=cache, page_table=table, lengths=lengths, counts=given, positions=positions))
        total = int(lengths.max())
        k, v = vgo.cache_read(cache, table, torch.zeros_like(lengths), total, lengths, dtype=F32)
        with torch.no_grad():
            qkv = wide.attn.qkv(wide.norm1(x.double())).reshape(2, count, 3, heads, d).permute(2, 0, 3, 1, 4)
            q = wide.attn.q_norm(qkv[0])
            if count > 1:
                q = wide.attn.apply_rope(q, q, (sin.double(), cos.double()))[0]
            else:
                q = torch.cat([wide.attn.apply_rope(q[:1], q[:1], (sin[7:8].double(), cos[7:8].double()))[0], q[1:]])
            scores = q @ k.double().transpose(-1, -2) / d ** 0.5
            scores = scores.masked_fill(torch.arange(total, device=device) >= lengths[:, None, None, None], -torch.inf)
            attended = (torch.softmax(scores, -1) @ v.double()).transpose(1, 2).reshape(2, count, dim)
            y = x.double() + wide.ls1(wide.attn.proj(attended))
            want = y + wide.ls2(wide.mlp(wide.norm2(y)))
        real = torch.ones(2, count, dtype=torch.bool, device=device)
        if given is not None:
            real = torch.arange(count, device=device) < given[:, None]
        assert (out.double() - want)[real].abs().max() <= step * want.abs().max()
        # What was stored are the format's numbers nearest to the block's values: off by at most one scale (half of the step
        # from 4 to 6, or 7 taken to 6), by two where the rounded block's largest crossed 7 and doubled it.
        first = (lengths - (count if given is None else given)).long()
        for b in range(2):
            stored = v[b, :, first[b]:lengths[b]].double().cpu()
            exact = qkv[2][b, :, :int(lengths[b] - first[b])].cpu()
            scale = 2.0 ** oracle.scale_exponents(exact.unflatten(-1, (-1, 32)).abs().amax(-1)).double()
            assert ((stored - exact).unflatten(-1, (-1, 32)).abs() <= 2.01 * scale[..., None] + step * exact.abs().max()).all()


def test_a_block_refuses(vgo, device):
    block = vgo.SelfAttentionBlock(128, 2).to(device)
    cache = vgo.PagedCache.empty(2, 2, 64, device=device)
    one = dict(cache=cache, page_table=int32([[0]], device), lengths=int32([4], device))
    x = torch.randn(1, 4, 128, device=device)
    with pytest.raises(RuntimeError, match="inference-only"):
        block.train()(x, cached=one)
    with pytest.raises(ValueError, match="neither"):
        block.eval()(x, attn_bias=dict(causal=True), cached=one)
    sin, cos = import_package("layers").rope_sincos(3, 3, 64, device=device)
    with pytest.raises(ValueError, match="positions"):
        block(x, (sin, cos), cached=one)
    assert not cache.data.any()


# ------------------------------------------------------------------------- surroundings ----
def scene(vgo, device, batch=2, tokens=700, heads=4, kv_heads=2, dim=64, n=1, dtype=BF16, page=64, masses=False, seed=0):
    """A filled cache, its table, and new tokens behind what it holds."""
    g = torch.Generator(device=device).manual_seed(seed)
    per = -(-(tokens + n) // page)
    cache = vgo.PagedCache.empty(batch * per, kv_heads, dim, page_size=page, masses=masses, device=device)
    table = torch.randperm(batch * per, generator=g, device=device).int().view(batch, per)
    draw = lambda h, m: torch.randn(batch, m, h, dim, generator=g, device=device).to(dtype).transpose(1, 2)
    k, v = draw(kv_heads, tokens), draw(kv_heads, tokens)
    vgo.cache_append(cache, k, v, table, torch.zeros(batch, dtype=torch.int32, device=device))
    starts = torch.full((batch,), tokens, dtype=torch.int32, device=device)
    return cache, table, starts, (draw(heads, n), draw(kv_heads, n), draw(kv_heads, n))


def step(vgo, cache, table, starts, new, **rules):
    q, k, v = new
    q = vgo.cache_append(cache, k, v, table, starts, q=q, rope=rules.pop("rope", None))
    return vgo.cached_attention(q, cache, table, starts + k.shape[2], **rules)


def tables(rows, dim, device):
    angle = torch.outer(torch.arange(rows, device=device), 100.0 ** (-torch.arange(dim // 2, device=device) / (dim // 2)))
    angle = torch.cat([angle, angle], 1)
    return angle.sin(), angle.cos()


@pytest.mark.parametrize("n", [1, 40, 300])
def test_captured_steps(vgo, device, n):
    """Two captured graphs of steps over two caches, replayed in turn on two streams beside eager work; lengths and inputs
    change in place between replays."""
    rope = tables(900, 64, device)
    scenes = [scene(vgo, device, n=n, seed=s) for s in range(2)]
    graphs, outs = [], []
    for cache, table, starts, new in scenes:
        step(vgo, cache, table, starts, new, rope=rope, causal=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(vgo, cache, table, starts, new, rope=rope, causal=True))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in scenes]
    for turn in range(4):
        for (cache, table, starts, new) in scenes:
            starts.fill_(700 - 13 * turn)
            for t in new:
                t.copy_(torch.randn(t.shape, device=device))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, (cache, table, starts, new) in zip(outs, scenes):
            got = out.clone()
            data = cache.data.clone()
            want = step(vgo, cache, table, starts, new, rope=rope, causal=True)
            assert torch.equal(got, want) and torch.equal(data, cache.data)
            torch.randn(1 << 20, device=device).sum()  # (eager work of another kind between the replays)


@pytest.mark.parametrize("n", [1, 300])
def test_streams_of_their_own(vgo, device, n):
    scenes = [scene(vgo, device, n=n, seed=s, tokens=3000) for s in range(4)]
    want = [step(vgo, *s) for s in scenes]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in scenes], []
    for s, stream in zip(scenes, streams):
        with torch.cuda.stream(stream):
            got.append([step(vgo, *s) for _ in range(3)])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_autocast(vgo, device, dtype):
    cache, table, starts, new = scene(vgo, device, dtype=F32, n=3)
    with torch.autocast("cuda", dtype=dtype):
        out = step(vgo, cache, table, starts, new)
    assert out.dtype == dtype
    assert torch.equal(out, step(vgo, cache, table, starts, [t.to(dtype) for t in new]))


def test_operators_by_name_and_traced(vgo, device):
    cache, table, starts, (q, k, v) = scene(vgo, device, n=5, masses=True)
    mass = torch.randn(2, 5, device=device)
    rope = tables(900, 64, device)

    def whole(q, k, v, data, page_mass, starts):
        q = torch.ops.vgo.cache_append(k, v, q, data, page_mass, table, starts, None, rope[0], rope[1], None, mass)
        k, v = torch.ops.vgo.cache_read(data, table, starts, None, 5, torch.bfloat16)
        return torch.ops.vgo.cached_attention(q, data, page_mass, table, starts + 5, None, True, 0.125), k, v

    plain = [t.clone() for t in (cache.data, cache.log_mass)]
    want = whole(q, k, v, plain[0], plain[1], starts)
    traced = [t.clone() for t in (cache.data, cache.log_mass)]
    got = torch.compile(whole, fullgraph=True)(q, k, v, traced[0], traced[1], starts)
    assert all(torch.equal(a, b) for a, b in zip((*want, *plain), (*got, *traced)))


def test_autograd_and_transforms(vgo, device):
    cache, table, starts, (q, k, v) = scene(vgo, device, n=5, masses=True)
    version = cache.data._version
    out = vgo.cache_append(cache, k, v, table, starts, q=q.clone().requires_grad_())
    assert out.requires_grad and cache.data._version > version and not cache.data.requires_grad
    with pytest.raises(RuntimeError, match="cache_append"):
        out.sum().backward()
    out = vgo.cached_attention(q.clone().requires_grad_(), cache, table, starts + 5)
    with pytest.raises(RuntimeError, match="cached_attention"):
        out.sum().backward()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: vgo.cached_attention(t, cache, table, starts + 5))(q[None])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: vgo.cache_append(cache, t, v, table, starts, q=q))(k[None])


def test_refusals(vgo, device):
    cache, table, starts, (q, k, v) = scene(vgo, device, n=5)
    rope = tables(900, 64, device)
    append = lambda **over: vgo.cache_append(*(over.get(n, x) for n, x in (("cache", cache), ("k", k), ("v", v), ("table", table),
                                                                         ("starts", starts))),
                                             **{n: x for n, x in over.items() if n not in ("cache", "k", "v", "table", "starts")})
    attend = lambda **over: vgo.cached_attention(*(over.get(n, x) for n, x in (("q", q), ("cache", cache), ("table", table),
                                                                             ("lengths", starts))),
                                                 **{n: x for n, x in over.items() if n not in ("q", "cache", "table", "lengths")})
    short, wide = cache._replace(data=cache.data[..., :100]), cache._replace(data=cache.data.int())
    masses = cache._replace(log_mass=torch.zeros(3, 64, device=device))
    for bad in (dict(k=k[:, :1]), dict(k=k[..., :32], v=v[..., :32]), dict(k=k.float()), dict(v=v[:, :, :4]), dict(q=q[:1]),
                dict(q=q.float()), dict(table=table.long()), dict(table=table[0]), dict(starts=starts.long()),
                dict(starts=starts[:1]), dict(counts=starts.float()), dict(cache=short), dict(cache=wide), dict(cache=masses),
                dict(positions=torch.zeros(2, 5, dtype=torch.int32, device=device)), dict(log_mass=torch.zeros(2, 5, device=device)),
                dict(rope=(rope[0], rope[1][:5])), dict(rope=(rope[0][:, :32], rope[1][:, :32])),
                dict(rope=rope, positions=torch.zeros(2, 4, dtype=torch.int32, device=device)), dict(k=k.double(), v=v.double()),
                dict(cache=cache._replace(data=cache.data.transpose(0, 1))),
                dict(table=torch.zeros(2, (1 << 24) + 1, dtype=torch.int32, device=device))):
        with pytest.raises((ValueError, RuntimeError)):
            append(**bad)
    for bad in (dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.double()), dict(table=table[:1]), dict(lengths=starts[:1]),
                dict(lengths=starts.long()), dict(counts=starts.float()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=1e9), dict(scale=1e-9), dict(cache=short), dict(cache=wide), dict(cache=masses)):
        with pytest.raises((ValueError, RuntimeError)):
            attend(**bad)
    for bad in (lambda: vgo.cache_read(cache, table, starts, -1), lambda: vgo.cache_read(cache, table, starts[:1], 3),
                lambda: vgo.cache_read(cache, table, starts, 3, dtype=torch.float64), lambda: vgo.cache_read(short, table, starts, 3)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


def test_empty_calls(vgo, device):
    cache, table, starts, (q, k, v) = scene(vgo, device, n=5)
    none = lambda *shape: torch.empty(shape, dtype=BF16, device=device)
    before = cache.data.clone()
    assert vgo.cache_append(cache, none(2, 2, 0, 64), none(2, 2, 0, 64), table, starts, q=none(2, 4, 0, 64)).shape == (2, 4, 0, 64)
    assert vgo.cache_append(cache, none(0, 2, 3, 64), none(0, 2, 3, 64), table[:0], starts[:0]) is None
    assert vgo.cache_read(cache, table, starts, 0)[0].shape == (2, 2, 0, 64)
    assert vgo.cached_attention(none(2, 4, 0, 64), cache, table, starts).shape == (2, 4, 0, 64)
    assert vgo.cached_attention(none(0, 4, 3, 64), cache, table[:0], starts[:0]).shape == (0, 4, 3, 64)
    assert torch.equal(before, cache.data)
    for n in (1, 200):  # no pages at all, and tables of nothing: nothing to attend to
        x = torch.randn(2, 4, n, 64, device=device).to(BF16)
        bare = vgo.PagedCache.empty(0, 2, 64, device=device)
        assert not vgo.cached_attention(x, bare, table, starts).any()
        assert not vgo.cached_attention(x, cache, table[:, :0], starts).any()
        vgo.cache_append(bare, x[:, :2], x[:, 2:], table, starts)
        assert not vgo.cache_read(bare, table, starts, 4)[0].any()


@pytest.mark.parametrize("n", [1, 130])
def test_offsets_past_32_bits(vgo, device, n):
    """Pages whose bytes lie past 2^32, in a cache and in its neighbours; queries whose strides pass it."""
    heads, page = 16, 1024
    each = heads * page // 32 * 34 * 64
    pages = (1 << 32) // each + 6
    cache = vgo.PagedCache.empty(pages, heads, 64, page_size=page, device=device)
    table = int32([[pages - 1, pages - 3], [pages - 2, 0]], device)
    g = torch.Generator(device=device).manual_seed(1)
    draw = lambda m: torch.randn(2, heads, m, 64, generator=g, device=device).to(BF16)
    k, v, zero = draw(1500), draw(1500), int32([0, 0], device)
    vgo.cache_append(cache, k, v, table, zero)
    small = vgo.PagedCache.empty(4, heads, 64, page_size=page, device=device)
    near = int32([[0, 1], [2, 3]], device)
    vgo.cache_append(small, k, v, near, zero)
    for a, b in zip(vgo.cache_read(cache, table, zero, 1500), vgo.cache_read(small, near, zero, 1500)):
        assert torch.equal(a, b)
    assert not cache.data[1:pages - 3].any()
    q, lengths = draw(n), int32([1500, 1400], device)
    assert torch.equal(vgo.cached_attention(q, cache, table, lengths), vgo.cached_attention(q, small, near, lengths))
    far = torch.empty(1 << 32, dtype=BF16, device=device).as_strided((2, heads, n, 64), ((1 << 31) + 64, 64, heads * 64, 1))
    far.copy_(q)
    assert torch.equal(vgo.cached_attention(far, small, near, lengths), vgo.cached_attention(q, small, near, lengths))


@pytest.mark.parametrize("n", [1, 300])
def test_another_device_or_a_current_one(vgo, device, n):
    """With one device: a tensor's own stays current; CPU lengths are refused."""
    cache, table, starts, new = scene(vgo, device, n=n)
    step(vgo, cache, table, starts, new)
    assert torch.cuda.current_device() == 0
    with pytest.raises(RuntimeError):
        vgo.cached_attention(new[0], cache, table, starts.cpu())
    with pytest.raises(RuntimeError):
        vgo.cache_append(cache, new[1], new[2], table.cpu(), starts)


@pytest.mark.parametrize("autocast", [False, True])
def test_a_block_with_gradients_enabled_and_captured(vgo, device, autocast):
    """Forward with gradients enabled gives what it gives without, and has no backward; a captured block's step replays."""
    torch.manual_seed(0)
    block = vgo.SelfAttentionBlock(128, 2, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device).eval()
    rope = import_package("layers").rope_sincos(4, 5, 64, device=device)
    table, lengths = int32([[1, 0], [2, 3]], device), int32([30, 25], device)
    x = torch.randn(2, 25, 128, device=device)
    caches = [vgo.PagedCache.empty(4, 2, 64, page_size=32, device=device) for _ in range(2)]
    steps = [dict(cache=c, page_table=table, lengths=lengths, causal=True) for c in caches]
    with torch.autocast("cuda", dtype=BF16, enabled=autocast):
        with torch.no_grad():
            want = block(x, rope, cached=steps[0])
        out = block(x, rope, cached=steps[1])
    assert (out - want).abs().max() <= (2.0 ** -4 if autocast else 2.0 ** -16) * want.abs().max()  # (other launches round elsewhere)
    with pytest.raises(RuntimeError):
        out.sum().backward()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, enabled=autocast, cache_enabled=False), torch.cuda.stream(stream):
        block(x, rope, cached=steps[0])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = block(x, rope, cached=steps[0])
    for turn in range(3):
        x.copy_(torch.randn_like(x))
        lengths.copy_(int32([30 + turn, 40 - turn], device))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad(), torch.autocast("cuda", dtype=BF16, enabled=autocast, cache_enabled=False):
            assert torch.equal(got, block(x, rope, cached=steps[0]))


def test_tangents_are_refused(vgo, device):
    """A tangent dropped would be a derivative of zero."""
    cache, table, starts, (q, k, v) = scene(vgo, device, n=5, masses=True)
    mass, rope = torch.zeros(2, 5, device=device), tables(900, 64, device)
    forward = torch.autograd.forward_ad
    before = cache.data.clone()
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))
        for call in (lambda: vgo.cached_attention(dual(q), cache, table, starts),
                     lambda: vgo.cache_append(cache, dual(k), v, table, starts), lambda: vgo.cache_append(cache, k, dual(v), table, starts),
                     lambda: vgo.cache_append(cache, k, v, table, starts, q=dual(q)),
                     lambda: vgo.cache_append(cache, k, v, table, starts, rope=(dual(rope[0]), rope[1])),
                     lambda: vgo.cache_append(cache, k, v, table, starts, log_mass=dual(mass))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        want = vgo.cached_attention(q, cache, table, starts)  # (without tangents as ever)
    assert torch.equal(before, cache.data) and torch.equal(want, vgo.cached_attention(q, cache, table, starts))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: vgo.cached_attention(t, cache, table, starts), (q,), (torch.ones_like(q),))


@pytest.mark.parametrize("n", [1, 40, 140])
def test_masses_at_any_float(vgo, device, n):
    """Masses that begin 4, 8 or 12 bytes past a multiple of 16: the same bits."""
    cache, table, starts, (q, k, v) = scene(vgo, device, n=n, masses=True)
    cache.log_mass.copy_(torch.randn(cache.log_mass.shape, generator=torch.Generator().manual_seed(3)))
    want = vgo.cached_attention(q, cache, table, starts)
    for at in (1, 2, 3):
        wide = torch.zeros(cache.log_mass.numel() + 4, device=device)
        view = wide[at:at + cache.log_mass.numel()].view(cache.log_mass.shape)
        view.copy_(cache.log_mass)
        assert torch.equal(want, vgo.cached_attention(q, cache._replace(log_mass=view), table, starts))
        vgo.cache_append(cache._replace(log_mass=view), k, v, table, starts, log_mass=torch.ones(2, n, device=device))
        assert (view != cache.log_mass).sum() == 2 * n and not wide[:at].any() and not wide[at + view.numel():].any()
