"""Shapes that the attention and the head norms refuse by name, whatever their defaults are made of."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("call,msg", [
    (lambda: net_ops.attention(*[meta(2, 3, 4, 0)] * 3), "omq_net::attention: heads"),
    (lambda: net_ops.attention_with_lse(*[meta(2, 3, 4, 0)] * 3), "omq_net::attention: heads"),
    (lambda: net_ops.attention_grad(*[meta(2, 3, 4, 0)] * 5, meta(2, 3, 4)),
     "omq_net::attention_grad: heads"),
    (lambda: net_ops.attention(*[meta()] * 3), "q must be"),
    (lambda: net_ops.head_norm_rotary(*[meta(2, 4, 8)] * 2, meta(2, 1, dtype=torch.int32),
                                      meta(dtype=torch.float64)), "frequencies must be"),
    (lambda: net_ops.head_norm_rotary_grad(*[meta(2, 4, 8)] * 4, meta(2, 1, dtype=torch.int32),
                                           meta(2, 2, dtype=torch.float64)), "frequencies must be"),
])
def test_refused(call, msg):
    with pytest.raises(RuntimeError, match=msg):
        call()
