"""Blocks whose attention has rules (`attn_bias`), with RoPE and prefix tokens, in inference and training."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import masked_attention as oracle
from tests.conftest import import_package

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [None, BF16, F16])
@pytest.mark.parametrize("prefix_tokens", [0, 5])
def test_block_with_rope_and_rules(vgo, device, monkeypatch, dtype, prefix_tokens):
    """Against the same block in 64 bits with a softmax over a dense bias: the fused LayerNorm and RoPE of inference, torch's
    operators of training, and the parameters' gradients."""
    layers = import_package("layers")
    torch.manual_seed(0)
    new_block = lambda: vgo.SelfAttentionBlock(128, 2, qkv_bias=True, use_qk_norm=True, init_values=0.5).to(device)
    block = new_block()
    rope = layers.rope_sincos(8, 12, 64, device=device)
    n = prefix_tokens + 96
    x = torch.randn(2, n, 128, device=device)
    table = torch.randn(32, 2, device=device, requires_grad=True)
    first = torch.tensor([20, 0], dtype=torch.int32, device=device)
    bias = dict(causal=True, prefix_lengths=first, bucket_table=table, score_cap=4.0)
    gap = torch.arange(n, device=device) - torch.arange(n, device=device)[:, None]
    ok = (gap <= 0) | (torch.arange(n, device=device) < first[:, None, None])

    wide, wide_table = new_block().double(), table.detach().double().requires_grad_()
    wide.load_state_dict(block.state_dict())
    dense = wide_table[oracle.bucket(gap.cpu(), 32, 128, True).to(device)].permute(2, 0, 1)

    def plain(q, k, v, **_):
        scores = torch.tanh(q @ k.transpose(-1, -2) / 8 / 4.0) * 4.0 + dense
        return torch.softmax(scores.masked_fill(~ok[:, None], -math.inf), -1) @ v

    with monkeypatch.context() as patch:
        patch.setattr(layers, "masked_attention", plain)
        ref = wide(x.double(), tuple(t.double() for t in rope), attn_bias=dict())
    parameters = lambda b, t: [t, b.attn.qkv.weight, b.norm1.weight, b.attn.q_norm.weight]
    expected = [ref, ref, *torch.autograd.grad(ref.sum(), parameters(wide, wide_table))]

    with torch.autocast("cuda", dtype=dtype or BF16, enabled=dtype is not None):
        out = block(x, rope, attn_bias=bias)
        grads = torch.autograd.grad(out.sum(), parameters(block, table))
        with torch.no_grad():
            inference = block.eval()(x, rope, attn_bias=bias)
    # About eight roundings in a row (norm, projection, q and k, P, output, projection, two of the MLP) of half a step
    # each, relative to the largest value and doubled by what the norms divide by: 16 half steps, 2^-4 in bf16.
    step = {None: 2.0 ** -16, BF16: 2.0 ** -4, F16: 2.0 ** -7}[dtype]
    for got, value in zip((out, inference, *grads), expected):
        assert (got.double() - value).abs().max() <= step * value.abs().max()
