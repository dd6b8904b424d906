"""Function transforms of the operators with gradients: what they have no derivative for is refused, never dropped."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests.test_gpu_masked_attention import F32, make

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused(vgo, device):
    """Tangents of any operand that the operators differentiate by, whether it requires grad or not."""
    q, k, v, rules, _ = make(device, F32, nq=20, nk=20, mass=True, slopes=True, buckets=8, distance=9)
    at = dict(q=q, k=k, v=v, **{n: rules.pop(n) for n in ("log_key_mass", "slopes", "bucket_table")})
    for grad_mode in (True, False):
        with torch.set_grad_enabled(grad_mode):
            for name, t in at.items():
                with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                    vgo.masked_attention(**{**at, name: forward_ad.make_dual(t, t)}, **rules)
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                vgo.relative_position_bias(forward_ad.make_dual(at["bucket_table"], at["bucket_table"]), 3, 3)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: vgo.masked_attention(t, k, v), (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: vgo.relative_position_bias(t, 3, 3), (at["bucket_table"],), (at["bucket_table"],))


def test_functional_gradients_are_refused(vgo, device):
    q, k, v, rules, _ = make(device, F32, nq=20, nk=20, buckets=8, distance=9)
    table = rules["bucket_table"]
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: vgo.masked_attention(q, k, v, bucket_table=t, max_distance=9).sum())(table)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: vgo.relative_position_bias(t, 3, 3, max_distance=9).sum())(table)


def test_values_under_vmap(vgo, device):
    tables = torch.randn(3, 8, 2, device=device)
    got = torch.func.vmap(lambda t: vgo.relative_position_bias(t, 5, 7, max_distance=9))(tables)
    for one, table in zip(got, tables):
        assert torch.equal(one, vgo.relative_position_bias(table, 5, 7, max_distance=9))
