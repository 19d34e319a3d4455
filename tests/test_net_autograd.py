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


def _calls(x):
    """The functions of net_ops on rows x [3, 8], each with its first result."""
    i, f, w = _meta(3, dtype=torch.int32), _meta(3), _meta(8)
    return {
        "token_embedding": lambda: net_ops.token_embedding(i, x),
        "token_embedding_grad": lambda: net_ops.token_embedding_grad(x, i, 4),
        "dropout": lambda: net_ops.dropout(x, 0.5, 1),
        "add_rms_norm": lambda: net_ops.add_rms_norm(x, None, w)[0],
        "add_rms_norm_fp8": lambda: net_ops.add_rms_norm_fp8(x, None, w)[1],
        "add_rms_norm_grad": lambda: net_ops.add_rms_norm_grad(x, None, x, w)[0],
        "clipped_policy_loss": lambda: net_ops.clipped_policy_loss(x, i, f, f)[0],
        "clipped_policy_loss_with_grad":
            lambda: net_ops.clipped_policy_loss_with_grad(x, i, f, f)[0],
    }


NAMES = list(_calls(None))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_raises(name, requires_grad):
    x = _meta(3, 8).requires_grad_(requires_grad)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, _meta(3, 8))
        with pytest.raises(NotImplementedError):
            _calls(dual)[name]()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: _calls(t)[name](), (_meta(3, 8),), (_meta(3, 8),))


@pytest.mark.parametrize("name", NAMES)
def test_backward_has_a_derivative_or_raises(name):
    x = _meta(3, 8).requires_grad_()
    out = _calls(x)[name]()
    assert out.requires_grad
    if name in ("token_embedding", "dropout", "add_rms_norm", "clipped_policy_loss"):
        out.sum().backward()
        assert x.grad.shape == x.shape
    else:  # (no derivative of their own)
        with pytest.raises(RuntimeError, match="not implemented"):
            out.sum().backward()
    with torch.no_grad():
        assert not _calls(x)[name]().requires_grad
