"""More of the attention's gradients on the GPU: parts of the keys with the whole row's out and lse.
Bounds as in test_gpu_attention.py."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops
from tests.test_gpu_attention import dense, inputs
from tests.test_gpu_net_ops import DTYPES, TINY, U, gen, within

pytestmark = pytest.mark.gpu


# ---- parts of the keys ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,heads,kv_heads,dim", [(90, 4, 2, 64), (5, 2, 1, 128), (130, 2, 2, 32)])
@pytest.mark.parametrize("cuts", [(0, 60, 100), (0, 300, 301, 700), (0, 40, 40, 500)])
def test_parts_of_the_keys(device, dtype, lq, heads, kv_heads, dim, cuts):
    """With the out and lse of all keys each part gives its own share: the parts' dq add up to the
    whole (each rounded), their dk and dv are the whole's."""
    lk = cuts[-1]
    q, k, v, go = inputs(gen(lq + lk), lq, lk, heads, kv_heads, dim, dtype)
    want, bound = dense(q, k, v, dim**-0.5, False, go)
    q, k, v, go = (t[None].to(device) for t in (q, k, v, go))
    out, lse = net_ops.attention_with_lse(q, k, v)
    parts = [net_ops.attention_grad(go, q, k[:, i:j].contiguous(), v[:, i:j].contiguous(), out, lse)
             for i, j in zip(cuts, cuts[1:])]
    within(torch.cat([p[1][0] for p in parts]), want["k"], bound["k"])
    within(torch.cat([p[2][0] for p in parts]), want["v"], bound["v"])
    each = [p[0][0].cpu().double() for p in parts]
    off = (sum(each) - want["q"]).abs()
    limit = bound["q"] + sum(U[dtype] * t.abs() + TINY[dtype] for t in each) * 1.01
    assert bool((off <= limit).all()), float((off / limit).max())
