"""The gradient of a bucket table where every sum is exact: whole numbers, so that one term left out, or taken twice, by
any lane, wave or part shows at once."""
from __future__ import annotations

import pytest
import torch

from oracle import masked_attention as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("nq, nk, buckets, rules", [
    (33, 5000, 32, {}), (130, 257, 32, {}), (300, 40, 64, dict(max_distance=400)), (1000, 1001, 32, {}),
    (70, 90, 32, dict(bidirectional=False)), (64, 2100, 16, dict(max_distance=1000)), (700, 1, 32, {}), (1, 700, 8, dict(max_distance=9)),
    (257, 300, 32, dict(query_start=-40)), (257, 300, 32, dict(query_start=250))])
def test_gradient_of_whole_numbers(vgo, device, dtype, nq, nk, buckets, rules):
    heads = 3
    g = torch.Generator().manual_seed(nq * 7 + nk)
    grad = torch.randint(-8, 9, (heads, nq, nk), generator=g).to(dtype)
    table = torch.randn(buckets, heads, generator=g).to(dtype).to(device).requires_grad_()
    bias = vgo.relative_position_bias(table, nq, nk, **rules)
    got, = torch.autograd.grad(bias, table, grad.to(device))
    wide = torch.zeros(buckets, heads, dtype=torch.float64, requires_grad=True)
    expected, = torch.autograd.grad(oracle.relative_position_bias(wide, nq, nk, **rules), wide, grad.double())
    assert 8 * nq * nk < 2 ** 24  # every partial sum is a whole number that fp32 holds
    assert torch.equal(got.cpu(), expected.to(dtype))
