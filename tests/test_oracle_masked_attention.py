"""The 64-bit masked attention: against torch's softmax, its gradients against differences, buckets against their
definition; and the host side of the operators (CPU only)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import masked_attention as oracle
from tests.conftest import import_package


def _inputs(b=2, h=4, hk=2, nq=7, nk=11, d=4):
    g = torch.Generator().manual_seed(5)
    draw = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)
    return draw(b, h, nq, d), draw(b, hk, nk, d), draw(b, hk, nk, d), draw(nk), draw(h).abs(), draw(8, h), draw(b, h, nq, d)


def _rules(b, nq, nk):
    g = torch.Generator().manual_seed(6)
    docs = torch.randint(0, 3, (b, nk), generator=g)
    return dict(causal=True, prefix_lengths=torch.tensor([2, 5][:b]), documents=docs[:, :nq], key_documents=docs,
                key_lengths=torch.tensor([nk, nk - 3][:b]), score_cap=1.5, max_distance=9, scale=0.7)


def test_plain_attention_is_torchs():
    q, k, v, *_ = _inputs(hk=4)
    out, _ = oracle.attention(q, k, v, dtype=torch.float32)
    ref = torch.softmax(q @ k.transpose(-1, -2) / 2.0, -1) @ v
    torch.testing.assert_close(out["out"], ref, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("name", ["q", "k", "v", "log_key_mass", "slopes", "bucket_table"])
def test_gradients_against_differences(name):
    q, k, v, mass, slopes, table, grad = _inputs()
    rules = _rules(2, 7, 11)
    at = dict(q=q, k=k, v=v, log_key_mass=mass, slopes=slopes, bucket_table=table)
    call = lambda t, g=None: oracle.attention(t["q"], t["k"], t["v"], t["log_key_mass"], slopes=t["slopes"],
                                              bucket_table=t["bucket_table"], grad=g, dtype=torch.float32, **rules)[0]
    got = call(at, grad)[name]
    step = 1e-6
    direction = torch.randn(at[name].shape, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
    up, down = (call({**at, name: at[name] + s * direction})["out"] for s in (step, -step))
    expected = ((up - down) / (2 * step) * grad).sum()
    assert abs((got * direction).sum() - expected) <= 1e-7 * max(1.0, abs(expected))


def test_rows_without_a_key():
    q, k, v, *_, grad = _inputs(b=1)
    res, _ = oracle.attention(q, k, v, grad=grad, documents=torch.full((1, 7), -1), key_documents=torch.zeros(1, 11),
                              dtype=torch.float32)
    assert all(not t.any() for t in res.values())


@pytest.mark.parametrize("buckets, distance, both", [(32, 128, True), (32, 128, False), (8, 9, True), (16, 500, True),
                                                     (2, 2, False), (64, 400, True), (4, 3, True)])
def test_bucket_starts(buckets, distance, both):
    """The host's starts against the definition; away from borders also against a logarithm in 64 bits."""
    starts = import_package("masked_attention")._bucket_starts(buckets, distance, both)
    gaps = torch.arange(-600, 601)
    n = gaps.abs() if both else (-gaps).clamp(min=0)
    counted = (n[:, None] >= torch.tensor(starts)).sum(1) + (buckets // 2 if both else 0) * (gaps > 0)
    expected = oracle.bucket(gaps, buckets, distance, both)
    assert torch.equal(counted if both else (n[:, None] >= torch.tensor(starts)).sum(1), expected)
    per = buckets // 2 if both else buckets
    e = per // 2
    grown = torch.log(n.clamp(min=1).double() / e) / math.log(distance / e) * (per - e)
    inside = (grown - grown.round()).abs() > 1e-9
    formula = torch.where(n < e, n, (e + grown.floor().long()).clamp(max=per - 1))
    assert torch.equal(formula[inside & (n >= e)], (expected % per if both else expected)[inside & (n >= e)])


def test_refusals_without_a_gpu():
    module = import_package("masked_attention")
    for wrong in ((1, 128, False), (3, 128, True), (2, 128, True), (32, 8, True), (258, 1000, False), (32, 1 << 21, True),
                  (32, 5000, True)):
        with pytest.raises(ValueError):
            module._bucket_starts(*wrong)
    q = torch.zeros(1, 1, 4, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        module.masked_attention(q, q, q)
    with pytest.raises(RuntimeError, match="GPU only"):
        module.relative_position_bias(torch.zeros(32, 2), 3, 3)


def _problem(lib_mod, **over):
    p = lib_mod.MaskedAttn(batch=1, heads=4, kv_heads=2, n_query=8, n_key=8, head_dim=64, scale=0.125, q=16, k=16, v=16)
    for s in (p.q_stride, p.k_stride, p.v_stride):
        s[:] = (2048, 512, 64)
    for name, value in over.items():
        setattr(p, name, value)
    return p


def test_c_entries_check_on_the_host():
    """Every refusal comes before a launch (and without a GPU); sizes of workspaces are refused short."""
    import ctypes
    lib_mod = import_package("_lib")
    lib = lib_mod.load()
    size = ctypes.c_size_t()
    starts = (ctypes.c_int32 * 3)(1, 5, 4)
    wrong = [dict(head_dim=32), dict(heads=3), dict(scale=0.0), dict(scale=math.inf), dict(score_cap=-1.0), dict(q=8),
             dict(k=None), dict(n_query=-1), dict(n_key=1 << 28), dict(prefix_lengths=16), dict(key_documents=16),
             dict(bucket_table=16, n_buckets=8, n_starts=3, bucket_starts=starts),
             dict(bucket_table=16, n_buckets=3, n_starts=2, bucket_starts=starts, bidirectional=1),
             dict(batch=1 << 20, heads=1 << 20)]
    for over in wrong:
        p = _problem(lib_mod, **over)
        assert lib.vgo_masked_attn_workspace(ctypes.byref(p), 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL, over
    p = _problem(lib_mod)
    p.q_stride[2] = 68
    assert lib.vgo_masked_attn_workspace(ctypes.byref(p), 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    p.q_stride[2] = 1 << 25
    assert lib.vgo_masked_attn_workspace(ctypes.byref(p), 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    p = _problem(lib_mod)
    assert lib.vgo_masked_attn_workspace(ctypes.byref(p), 7, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    assert lib.vgo_masked_attn_workspace(None, 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    g = lib_mod.MaskedAttnGrads(out=16, grad_out=16, lse=16, dq=16)
    for s in (g.out_stride, g.grad_out_stride, g.dq_stride):
        s[:] = (2048, 512, 64)
    assert lib.vgo_masked_attn_grad_workspace(ctypes.byref(p), ctypes.byref(g), 1, ctypes.byref(size)) == lib_mod.VGO_OK
    assert size.value > 0
    assert lib.vgo_masked_attn_grad(ctypes.byref(p), ctypes.byref(g), 1, 16, size.value - 1, None) == lib_mod.VGO_EWORKSPACE
    assert lib.vgo_masked_attn_grad(ctypes.byref(p), ctypes.byref(g), 1, None, 0, None) == lib_mod.VGO_EWORKSPACE
    for name in ("d_log_mass", "d_slopes", "d_table", "dk"):
        more = lib_mod.MaskedAttnGrads.from_buffer_copy(g)
        setattr(more, name, 16)
        assert lib.vgo_masked_attn_grad_workspace(ctypes.byref(p), ctypes.byref(more), 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    good = (ctypes.c_int32 * 3)(1, 2, 3)
    bias = lambda **o: lib.vgo_position_bias(*{**dict(table=16, buckets=8, heads=2, starts=good, n=3, both=1, start=0, nq=4,
                                                       nk=4, out=None, dtype=1, stream=None), **o}.values())
    assert bias() == lib_mod.VGO_EINVAL and bias(starts=starts, out=16) == lib_mod.VGO_EINVAL
    assert bias(buckets=7, out=16) == lib_mod.VGO_EINVAL and bias(nq=-1, out=16) == lib_mod.VGO_EINVAL
    assert lib.vgo_position_bias_grad(16, 8, 2, good, 3, 1, 0, 4, 4, 16, 1, None, 0, None) == lib_mod.VGO_EWORKSPACE
