"""What the masked attention takes and refuses, on the host (CPU only)."""
from __future__ import annotations

import ctypes

import pytest

from tests.conftest import import_package
from tests.test_oracle_masked_attention import _problem


def workspace(**over):
    """(status, bytes) of the forward's workspace for a small problem with these fields set."""
    lib_mod = import_package("_lib")
    size = ctypes.c_size_t()
    problem = _problem(lib_mod, **over)
    return lib_mod.load().vgo_masked_attn_workspace(ctypes.byref(problem), 1, ctypes.byref(size)), size.value


@pytest.mark.parametrize("sizes", [dict(n_query=0), dict(n_key=0), dict(n_query=0, n_key=0), dict(batch=0)])
@pytest.mark.parametrize("side", ["query_documents", "key_documents"])
def test_documents_of_an_empty_side_may_be_null(sizes, side):
    lib_mod = import_package("_lib")
    assert workspace(**{side: 16}, **sizes)[0] == lib_mod.VGO_OK
    assert workspace(**{side: 16})[0] == lib_mod.VGO_EINVAL


def test_rules_beside_a_token_plan_are_refused():
    """In attention itself as in the module's forward, which hands them on."""
    import torch
    attention = import_package("layers").SelfAttention(128, 2).eval()
    qkv = torch.zeros(1, 5, 384)
    for call in (lambda: attention.compute_attention(qkv, attn_bias=dict(causal=True), token_plan=object()),
                 lambda: attention._forward_merged(torch.zeros(1, 5, 128), dict(causal=True), None, object()),
                 lambda: attention(torch.zeros(1, 5, 128), attn_bias=dict(causal=True), token_plan=object())):
        with pytest.raises(ValueError, match="token plan"):
            call()


def test_more_work_groups_than_a_grid_has_threads_for():
    """Refused on the host, not left to the launch: a grid's threads are counted in 32 bits."""
    lib_mod = import_package("_lib")
    lib = lib_mod.load()
    sizes = dict(heads=16, kv_heads=16, n_query=1, n_key=1)
    assert workspace(batch=1 << 20, **sizes)[0] == lib_mod.VGO_EINVAL
    assert workspace(batch=(1 << 20) - 1, **sizes)[0] == lib_mod.VGO_OK
    grads = lib_mod.MaskedAttnGrads(out=16, grad_out=16, lse=16, dq=16)
    size = ctypes.c_size_t()
    for batch, status in ((1 << 20, lib_mod.VGO_EINVAL), (1 << 18, lib_mod.VGO_OK)):
        problem = _problem(lib_mod, batch=batch, **sizes)
        assert lib.vgo_masked_attn_grad_workspace(ctypes.byref(problem), ctypes.byref(grads), 1, ctypes.byref(size)) == status
    starts = (ctypes.c_int32 * 1)(1)
    many = lambda n_query: lib.vgo_position_bias_grad(16, 4, 16, starts, 1, 1, 0, n_query, 1, 16, 1, None, 0, None)
    assert many(1 << 25) == lib_mod.VGO_EINVAL and "too many rows" in lib_mod.last_error()
    assert many(1 << 20) == lib_mod.VGO_EWORKSPACE
    assert lib.vgo_position_bias(16, 4, 1 << 24, starts, 1, 1, 0, 1, 1, 16, 1, None) == lib_mod.VGO_EINVAL
