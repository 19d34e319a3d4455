"""More of the log-probabilities on the GPU: rows whose legal tokens lie in one wave's part, and
entropy weights of any size.  Bounds as in test_gpu_logprobs.py."""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_logprobs import bounds
from tests.test_gpu_net_ops import DTYPES, gen, randn, within

pytestmark = pytest.mark.gpu


def gradients(device, z, tokens, legal, a, b):
    """By the fused call and by autograd."""
    z, tokens, legal, a, b = (None if t is None else t.to(device) for t in (z, tokens, legal, a, b))
    both = net_ops.token_logprobs_with_grad(z, tokens, a, b, legal)[2]
    x = z.clone().requires_grad_()
    auto = net_ops.token_logprobs(x, tokens, legal)
    torch.autograd.backward(auto[:2], (a, b))
    return both, x.grad


def far_rows(vocab, dtype, level, at):
    """Nine legal tokens from `at` on, about `level`; one row by a mask over NaN, one by -infinity."""
    g = gen(vocab + at)
    z = torch.full((2, vocab), math.nan)
    z[1] = -math.inf
    z[:, at:at + 9] = level + randn(g, 2, 9)
    legal = torch.zeros(2, vocab, dtype=torch.bool)
    legal[0, at:at + 9] = True
    legal[1] = True
    return (z.to(dtype), torch.tensor([at + 4, at]), legal, torch.tensor([1.0, -2.0]),
            torch.tensor([0.5, 0.1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,at", [(40, 3), (1025, 700), (2000, 5), (3000, 1700), (4672, 40),
                                      (8192, 8000), (12000, 600), (16384, 16300), (20_000, 12345)])
@pytest.mark.parametrize("level", [-95.0, -200.0, -30000.0, 200.0])
def test_legal_tokens_of_one_wave(device, dtype, vocab, at, level):
    """The other waves have no logit that counts, whatever the size of those that do."""
    z, tokens, legal, a, b = far_rows(vocab, dtype, level, at)
    want = net_ref.token_logprobs(z, tokens, legal, 0, a, b)[4]
    e_grad = bounds(z.nan_to_num(0.0, 0.0, -math.inf), legal, tokens, a, b)[2]
    for grad in gradients(device, z, tokens, legal, a, b):
        within(grad, want, e_grad.nan_to_num(0.0))
        assert not bool(grad.cpu()[0][~legal[0]].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 600, 3000, 8192, 16384, 20_000])
@pytest.mark.parametrize("weight", [1e8, 1e9, -3e9, 1e20, 1e30])
def test_large_entropy_weights(device, dtype, vocab, weight):
    """0 at tokens that are not legal, or of probability 0 (a third are -1e30, a third are not
    legal)."""
    g = gen(vocab)
    z = randn(g, 4, vocab)
    z[:, ::3] = -1e30
    legal = torch.ones(4, vocab, dtype=torch.bool)
    legal[:, 1::3] = False
    z[:, 1::3] = math.nan
    z = z.to(dtype)
    tokens = torch.tensor([2, 5, -1, 3])
    a, b = randn(g, 4), torch.full((4,), weight)
    want = net_ref.token_logprobs(z, tokens, legal, 0, a, b)[4]
    e_grad = bounds(z.nan_to_num(0.0), legal, tokens, a, b)[2]
    for grad in gradients(device, z, tokens, legal, a, b):
        # (where p is 0 the bound's allowance for p grows with the logit; the gradient is 0)
        grad = grad.cpu()
        assert not bool(grad[:, ::3][tokens[:, None].expand(4, vocab)[:, ::3] !=
                                     torch.arange(vocab)[::3]].any())
        assert not bool(grad[:, 1::3].any())
        within(grad[:, 2::3], want[:, 2::3], e_grad[:, 2::3])
