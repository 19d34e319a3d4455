"""More of the log-probabilities on the GPU: rows whose legal tokens lie in one wave's part, entropy
weights of any size, and long rows that are many.  Bounds as in test_gpu_logprobs.py."""
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


def plain(z, tokens, legal, top, a, b):
    """net_ref.token_logprobs of finite legal logits, all rows at once."""
    zl = z.double().masked_fill(~legal, -math.inf)
    logq = torch.log_softmax(zl, 1)
    p = logq.exp()
    plogp = torch.where(legal, p * logq.masked_fill(~legal, 0.0), 0.0)
    entropy = -plogp.sum(1)
    given = (tokens >= 0) & (tokens < z.shape[1])
    at = torch.where(given, tokens, 0)[:, None]
    given &= legal.gather(1, at)[:, 0]
    logp = torch.where(given, logq.gather(1, at)[:, 0], 0.0)
    order = torch.sort(zl, dim=1, descending=True, stable=True)[1][:, :top]
    a = torch.where(given, a.double(), 0.0)[:, None]
    grad = -a * p - b.double()[:, None] * (plogp + p * entropy[:, None])
    grad.scatter_add_(1, at, a)
    return logp, entropy, logq.gather(1, order), order, grad


def test_the_rows_at_once_are_the_definition():
    g = gen(2)
    z, tokens = randn(g, 6, 50, dtype=torch.bfloat16), torch.tensor([0, 7, -1, 50, 49, 3])
    legal = torch.rand(6, 50, generator=g) < 0.7
    a, b = randn(g, 6), randn(g, 6)
    args = (z, tokens, legal, 5, a, b)
    for x, y in zip(plain(*args), net_ref.token_logprobs(*args)):
        assert torch.allclose(x.double(), y.double(), atol=1e-12)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(520, 16392), (513, 20_001), (1100, 16400)])
def test_many_long_rows(device, dtype, rows, vocab):
    """Rows that a workgroup of 256 threads reads, with a mask, ties among the best and gradients."""
    g = gen(rows + vocab)
    z = (randn(g, rows, vocab) * 4).round().div(2).to(dtype)  # (halves: many are alike)
    z[::5] = randn(g, len(range(0, rows, 5)), vocab, dtype=dtype)
    tokens = torch.randint(-1, vocab + 1, (rows,), generator=g)
    legal = torch.rand(rows, vocab, generator=g) < 0.8
    z[7, 100:] = 0.5  # (more ties than a row's list of candidates holds)
    z[7, :100] = -3.0
    a, b = randn(g, rows), randn(g, rows, scale=0.1)
    want = plain(z, tokens, legal, 32, a, b)
    e_logp, e_h, e_grad, _ = bounds(z, legal, tokens, a, b)
    zd, td, ld = (t.to(device) for t in (z.masked_fill(~legal, math.nan), tokens, legal))
    logp, entropy, top_logp, top_tokens = net_ops.token_logprobs(zd, td, ld, 32)
    assert torch.equal(top_tokens.cpu(), want[3])
    within(top_logp, want[2], e_logp[:, None].expand(-1, 32))
    both = net_ops.token_logprobs_with_grad(zd, td, a.to(device), b.to(device), ld)
    within(both[2], want[4], e_grad)
    for lp, h in ((logp, entropy), both[:2]):
        within(lp, want[0], e_logp)
        within(h, want[1], e_h)
