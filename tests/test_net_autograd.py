"""What the policy network's operators leave for automatic differentiation, on meta tensors: shapes
of empty batches, and errors where there is no derivative."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("shape", [(0, 8), (3, 0, 8), (2, 8)])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_norm_of_an_empty_batch(shape, with_residual, p):
    x, w = _meta(*shape).requires_grad_(), _meta(8).requires_grad_()
    res = _meta(*shape).requires_grad_() if with_residual else None
    y, h = net_ops.add_rms_norm(x, res, w, p=p)
    assert y.shape == h.shape == x.shape
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    assert res is None or res.grad.shape == x.shape
