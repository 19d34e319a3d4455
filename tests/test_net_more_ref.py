"""The definitions in 64 bits of the head norms, the attention and the log-probabilities
(oracle/net_ref.py) against torch's own operators and derivatives, and by known answers."""
import math

import pytest
import torch

from oracle import net_ref


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_rotation(interleaved, weighted):
    g = gen(1)
    x = torch.randn(5, 3, 11, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.rand(11, generator=g, dtype=torch.float64).requires_grad_() if weighted else None
    pos = torch.randint(-9, 9, (5, 2), generator=g)
    f = torch.rand(4, generator=g, dtype=torch.float64)
    args = (pos, f, w, 1e-3, (1, 3), interleaved)
    out = net_ref.head_norm_rotary(x, *args)
    n = x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-3) * w
    axis = torch.tensor([0, 1, 1, 1])
    t = torch.polar(torch.ones(5, 4).double(), pos[:, axis] * f)[:, None]
    one, two = ((0, 2, 4, 6), (1, 3, 5, 7)) if interleaved else ((0, 1, 2, 3), (4, 5, 6, 7))
    z = torch.complex(n[..., one], n[..., two]) * t
    assert torch.allclose(out[..., one], z.real, atol=1e-12)
    assert torch.allclose(out[..., two], z.imag, atol=1e-12)
    assert torch.equal(out[..., 8:], n[..., 8:])
    go = torch.randn(out.shape, generator=g, dtype=torch.float64)
    out.backward(go)
    gx, gw = net_ref.head_norm_rotary_grad(go, x.detach(), *args)
    assert torch.allclose(gx, x.grad, atol=1e-12)
    assert gw is None if w is None else torch.allclose(gw, w.grad, atol=1e-12)


def test_a_quarter_turn():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0]]])
    f = torch.tensor([math.pi / 2, 0.0], dtype=torch.float64)
    for inter, want in ((False, [-3, 2, 1, 4, 5]), (True, [-2, 1, 3, 4, 5])):
        got = net_ref.head_norm_rotary(x, torch.tensor([[1]]), f, None, 0.0, (2,), inter)
        assert torch.allclose(got[0, 0], torch.tensor(want).double(), atol=1e-12)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [(4, 4), (2, 7), (7, 3), (1, 1)])
def test_attention(causal, lq, lk):
    g = gen(lq + lk)
    q = torch.randn(lq, 4, 6, generator=g, dtype=torch.float64).requires_grad_()
    k, v = (torch.randn(lk, 2, 6, generator=g, dtype=torch.float64).requires_grad_()
            for _ in range(2))
    go = torch.randn(lq, 4, 6, generator=g, dtype=torch.float64)
    out, lse, gq, gk, gv = net_ref.attention(q.detach(), k.detach(), v.detach(), 0.3, causal, go)
    kk, vv = (t.repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))
    s = 0.3 * q.transpose(0, 1) @ kk.transpose(1, 2)
    hidden = torch.ones(lq, lk, dtype=torch.bool).triu(lk - lq + 1) & causal
    p = torch.softmax(s.masked_fill(hidden, -1e300), 2)
    p = p * (~hidden).any(1)[None, :, None]  # (a query that sees nothing)
    want = (p @ vv).transpose(0, 1)
    want.backward(go)
    assert torch.allclose(out, want, atol=1e-12)
    live = (~hidden).any(1)
    assert torch.allclose(lse[live], torch.logsumexp(s.masked_fill(hidden, -math.inf), 2).t()[live])
    assert bool((lse[~live] == -math.inf).all())
    for a, b in ((gq, q.grad), (gk, k.grad), (gv, v.grad)):
        assert torch.allclose(a, b, atol=1e-12)


def test_attention_of_one_key_is_its_value():
    v = torch.tensor([[[3.0, -1.0]]])
    out, lse = net_ref.attention(torch.ones(2, 3, 2), torch.ones(1, 1, 2), v, 2.0, False)
    assert torch.equal(out, v.double().expand(2, 3, 2)) and bool((lse == 4.0).all())


@pytest.mark.parametrize("masked", [False, True])
def test_logprobs(masked):
    g = gen(3)
    z = torch.randn(6, 9, generator=g, dtype=torch.float64).requires_grad_()
    legal = torch.rand(6, 9, generator=g) < 0.6 if masked else None
    tokens = torch.randint(0, 9, (6,), generator=g)
    if masked:
        legal.scatter_(1, tokens[:, None], True)
    tokens[2] = -1
    a, b = torch.randn(6, generator=g), torch.randn(6, generator=g)
    logp, entropy, top_logp, top_tokens, grad = net_ref.token_logprobs(z.detach(), tokens, legal, 3,
                                                                       a, b)
    zl = z if legal is None else z.masked_fill(~legal, -1e30)
    logq = torch.log_softmax(zl, 1)
    h = torch.distributions.Categorical(logits=zl).entropy()
    lp = logq.gather(1, tokens.clamp(min=0)[:, None])[:, 0] * (tokens >= 0)
    assert torch.allclose(logp, lp) and torch.allclose(entropy, h, atol=1e-6)
    (a * lp + b * -(logq.exp() * logq).sum(1)).sum().backward()
    assert torch.allclose(grad, z.grad, atol=1e-12)
    values, index = torch.topk(logq, 3, 1)
    fine = values > -1e20
    assert torch.equal(top_tokens[fine], index[fine]) and torch.allclose(top_logp[fine], values[fine])
    assert bool((top_tokens[~fine] == -1).all())


def test_logprobs_by_hand():
    z = torch.tensor([[0.0, 0.0, -math.inf, 0.0], [1.0, 2.0, 3.0, 4.0]])
    legal = torch.tensor([[True, True, True, True], [False] * 4])
    logp, entropy, top_logp, top, _ = net_ref.token_logprobs(z, torch.tensor([3, 0]), legal, 4)
    assert float(logp[0]) == pytest.approx(-math.log(3)) and float(logp[1]) == 0
    assert float(entropy[0]) == pytest.approx(math.log(3)) and float(entropy[1]) == 0
    assert top.tolist() == [[0, 1, 3, -1], [-1] * 4] and float(top_logp[0, 3]) == -math.inf
