"""The dense relative position bias and the gradient of its table."""
from __future__ import annotations

import pytest
import torch

from oracle import masked_attention as oracle

pytestmark = pytest.mark.gpu

CASES = [(1, 1, 32, 1, {}), (1, 700, 32, 8, {}), (5, 3, 8, 2, dict(max_distance=9)), (130, 257, 32, 3, {}),
         (64, 64, 16, 4, dict(max_distance=500)), (300, 40, 64, 2, dict(max_distance=400)), (33, 5000, 32, 1, {}),
         (70, 90, 32, 2, dict(bidirectional=False)), (20, 30, 32, 2, dict(query_start=-500)),
         (20, 30, 32, 2, dict(query_start=900)), (40, 300, 2, 2, dict(bidirectional=False, max_distance=2)),
         (50, 60, 32, 2, dict(max_distance=2048)), (0, 7, 32, 2, {}), (7, 0, 32, 2, {})]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("nq, nk, buckets, heads, rules", CASES)
def test_bias_and_gradient(vgo, device, dtype, nq, nk, buckets, heads, rules):
    g = torch.Generator().manual_seed(nq + nk)
    table = torch.randn(buckets, heads, generator=g).to(dtype)
    grad = torch.randn(heads, nq, nk, generator=g).to(dtype)
    leaf = table.to(device).requires_grad_()
    bias = vgo.relative_position_bias(leaf, nq, nk, **rules)
    expected = oracle.relative_position_bias(table, nq, nk, **rules)
    assert bias.dtype == dtype and torch.equal(bias.detach().cpu(), expected)
    got, = torch.autograd.grad(bias, leaf, grad.to(device))
    wide = table.double().requires_grad_()
    ref, = torch.autograd.grad(oracle.relative_position_bias(wide, nq, nk, **rules), wide, grad.double())
    size = torch.zeros(buckets, heads, dtype=torch.float64)
    size, = torch.autograd.grad(oracle.relative_position_bias(wide, nq, nk, **rules), wide, grad.double().abs())
    # Half a step of fp32 for every term of a sum, and of the type for its rounding.
    bound = nq * nk * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * ref.abs()
    assert ((got.double().cpu() - ref).abs() <= bound + 1e-7).all()
    again, = torch.autograd.grad(vgo.relative_position_bias(leaf, nq, nk, **rules), leaf, grad.to(device))
    assert torch.equal(got, again)


def test_strided_and_misaligned(vgo, device):
    """A table and a gradient that are views, rows that start off 16 bytes."""
    table = torch.randn(2, 32, 2, device=device).bfloat16().permute(2, 1, 0)[1].requires_grad_()  # [32, 2], strided
    bias = vgo.relative_position_bias(table, 37, 61)
    assert torch.equal(bias.detach().cpu(), oracle.relative_position_bias(table.detach().cpu(), 37, 61))
    grad = torch.randn(2, 61, 37, device=device).bfloat16().transpose(1, 2)
    got, = torch.autograd.grad(bias, table, grad)
    ref, = torch.autograd.grad(vgo.relative_position_bias(table, 37, 61), table, grad.contiguous())
    assert torch.equal(got, ref)


def test_refusals(vgo, device):
    table = torch.randn(32, 2, device=device)
    for call in (lambda: vgo.relative_position_bias(table[0], 3, 3), lambda: vgo.relative_position_bias(table.double(), 3, 3),
                 lambda: vgo.relative_position_bias(table, -1, 3), lambda: vgo.relative_position_bias(table[:31], 3, 3),
                 lambda: vgo.relative_position_bias(table, 3, 3, max_distance=7),
                 lambda: vgo.relative_position_bias(table, 3, 3, max_distance=9000),
                 lambda: vgo.relative_position_bias(table, 3, 1 << 28),
                 lambda: vgo.relative_position_bias(table, 3, 3, query_start=1 << 40)):
        with pytest.raises(ValueError):
            call()
