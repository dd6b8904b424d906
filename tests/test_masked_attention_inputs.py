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
