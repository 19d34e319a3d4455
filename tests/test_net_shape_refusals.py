"""Shapes and scales that the attention and the head norms refuse by name."""
import pytest
import torch

from omoknuni_quantum_amd import _lib, net_ops


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


def test_scales_whose_product_with_log2_e_is_not_finite():
    q = meta(2, 3, 4, 8)
    assert net_ops.attention(q, q, q, scale=2.0**127).shape == q.shape
    for scale in (2.5e38, 3.4e38, 1e39):
        with pytest.raises(RuntimeError, match="above 0"):
            net_ops.attention(q, q, q, scale=scale)
    lib, one = _lib.load_net(), 4096
    a = _lib.OmqAttentionArgs(sequences=2, q_len=5, k_len=7, q=one, k=one, v=one, q_heads=4,
                              k_heads=2, dim=32, dtype=0, scale=2.0**127)
    assert lib.omq_attention_grad_workspace(a) > 0
    a.scale = 2.5e38
    assert lib.omq_attention_grad_workspace(a) == _lib.OMQ_E_ARG
