"""Log-probabilities of tokens on the GPU against their definition in 64 bits (oracle/net_ref.py).

Tolerances, u = 2^-24, of rows of V tokens, x = z - max z, E the mean under the row's distribution.
A thread adds at most 16 + V / 1024 exponentials in a row (each after at most as many rescalings)
and 20 joins follow; an exponential is off by (|x| + 2) u, relative.  So s is off by
S = (36 + V / 512 + E|x| + 4) u relative, logp and log s by S + 2 u + 2^-25 and their rounding, and
the entropy by S (1 + E|x|) + u E x^2 + 8 u (1 + E|x|).  A gradient's element
p (a + b (log p + H)) is off by p (|a| + |b| |log p + H|) (S + (|x| + 8) u) +
|b| p (off of log p + off of H + 4 u (|x| + log V)), and the given token's has a S (1 - p) more.
The instruction of 2^x gives 0 in place of results below 2^-126, the least normal number: p, which
is such a result over s >= 1, may be off by 2^-126 for that, whatever its size, and the element by
2^-126 (|a| + |b| |log p + H|)."""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_net_ops import DTYPES, gen, randn, strided, u, within

pytestmark = pytest.mark.gpu


def bounds(z, legal, tokens, a, b):
    z = z.double()
    if legal is not None:
        z = z.masked_fill(~legal, -math.inf)
    vocab = z.shape[1]
    live = (z > -math.inf).any(1)
    logq = torch.log_softmax(z, 1)
    p = torch.where(live[:, None], logq.exp(), 0.0)
    x = torch.where(p > 0, (z.amax(1, keepdim=True) - z), 0.0)
    logq = torch.where(p > 0, logq, 0.0)
    h = -(p * logq).sum(1)
    ex, exx = (p * x).sum(1), (p * x * x).sum(1)
    s = (40 + vocab / 512 + ex) * u
    e_logp = s + 4 * u
    e_h = s * (1 + ex) + u * exx + 8 * u * (1 + ex)
    a, b = a.double().abs()[:, None], b.double().abs()[:, None]
    away = (logq + h[:, None]).abs()
    grad = p * (a + b * away) * (s[:, None] + (x + 8) * u) + \
        b * p * ((e_logp + e_h)[:, None] + 4 * u * (x + math.log(vocab)))
    grad = grad + 2.0**-126 * (a + b * (x + h[:, None] + math.log(vocab)))
    at = tokens.long().clamp(0, vocab - 1)[:, None]
    grad.scatter_add_(1, at, a * (s[:, None] + 4 * u) * (1 - p.gather(1, at)))
    return e_logp, e_h, grad, live


def rows_of(seed, rows, vocab, dtype, masked):
    g = gen(seed)
    z = randn(g, rows, vocab, dtype=dtype, scale=2.0)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    legal = None
    if masked:
        legal = torch.rand(rows, vocab, generator=g) < torch.rand(rows, 1, generator=g)
        legal.scatter_(1, tokens[:, None], True)
        legal[::7] = False
        tokens[3::7] = (tokens[3::7] + 1) % vocab  # (perhaps not legal)
        z[~legal] = float("nan")
    tokens[2::9] = -1
    if rows > 5:
        tokens[5] = vocab
    return z, tokens, legal, randn(g, rows), randn(g, rows, scale=0.1)


def check(device, z, tokens, legal, a, b, top, extra=3):
    zd = strided(z, extra, device)
    ld = None if legal is None else strided(legal, extra, device)
    td = tokens.to(device)
    want = net_ref.token_logprobs(z, tokens, legal, top, a, b)
    e_logp, e_h, e_grad, live = bounds(z.nan_to_num(0.0) if legal is not None else z, legal, tokens,
                                       a, b)
    logp, entropy, top_logp, top_tokens = net_ops.token_logprobs(zd, td, ld, top)
    assert torch.equal(top_tokens.cpu(), want[3])
    within(top_logp, want[2], e_logp[:, None].expand(-1, top))
    both = net_ops.token_logprobs_with_grad(zd, td, a.to(device), b.to(device), ld)
    x = zd.detach().clone().requires_grad_()
    auto = net_ops.token_logprobs(x, td, ld, top)
    ((auto[0] * a.to(device)) + (auto[1] * b.to(device))).sum().backward()
    for lp, h, grad in ((logp, entropy, None), both, (auto[0].detach(), auto[1].detach(), x.grad)):
        within(lp, want[0], e_logp)
        within(h, want[1], e_h)
        if grad is not None:
            within(grad, want[4], e_grad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (9, 5, 8), (64, 225, 5), (10, 361, 0),
                                            (8, 512, 32), (8, 513, 3), (7, 1025, 8), (6, 2048, 20),
                                            (6, 4095, 32), (5, 4672, 8), (3, 8200, 7),
                                            (3, 16384, 32), (3, 16391, 9), (2, 40_000, 32)])
def test_rows(device, dtype, masked, rows, vocab, top):
    check(device, *rows_of(rows + vocab, rows, vocab, dtype, masked), top)


@pytest.mark.parametrize("vocab", [30, 512, 600, 4096, 9000, 20_000])
@pytest.mark.parametrize("kind", ["equal", "two values", "falling", "lowest", "signed zeros"])
def test_ties(device, vocab, kind):
    """Equal logits go to the lowest index, however many there are."""
    g = gen(vocab)
    z = torch.zeros(3, vocab)
    if kind == "two values":
        z = torch.randint(0, 2, (3, vocab), generator=g).float()
    elif kind == "falling":
        z = -torch.arange(3 * vocab).view(3, vocab).float() / 64
    elif kind == "lowest":
        z[:, vocab // 3:] = torch.finfo(torch.float32).min
        z[1] = torch.finfo(torch.float32).min
    elif kind == "signed zeros":
        z = torch.where(torch.rand(3, vocab, generator=g) < 0.5, -0.0, 0.0)
    tokens = torch.tensor([0, 1, vocab // 2])
    for top in (1, 17, 32):
        check(device, z, tokens, None, torch.ones(3), torch.ones(3), top, extra=0)


@pytest.mark.parametrize("vocab", [40, 700, 3000, 8192, 20_000])
def test_probabilities_of_zero_and_no_legal_token(device, vocab):
    g = gen(vocab)
    z = randn(g, 5, vocab)
    z[0] = -math.inf
    z[1, 1:] = -math.inf
    z[2, ::2] = -math.inf
    z[3, :vocab - 3] = -math.inf
    legal = torch.ones(5, vocab, dtype=torch.bool)
    legal[4] = False
    tokens = torch.tensor([0, 0, 2, vocab - 1, 1])  # (row 2's has probability 0)
    a, b = randn(g, 5), randn(g, 5)
    want = net_ref.token_logprobs(z, tokens, legal, 6, a, b)
    assert float(want[0][2]) == -math.inf and float(want[0][1]) == 0
    e_logp, e_h, e_grad, _ = bounds(z, legal, tokens, a, b)
    dev = [t.to(device) for t in (z, tokens, legal)]
    logp, entropy, top_logp, top_tokens = net_ops.token_logprobs(*dev, 6)
    assert torch.equal(top_tokens.cpu(), want[3])
    within(top_logp, want[2], e_logp[:, None].expand(-1, 6).nan_to_num(0.0))
    x = dev[0].clone().requires_grad_()
    auto = net_ops.token_logprobs(x, *dev[1:])
    torch.autograd.backward(auto[:2], (a.to(device), b.to(device)))
    both = net_ops.token_logprobs_with_grad(*dev[:2], a.to(device), b.to(device), dev[2])
    for lp, h, grad in ((logp, entropy, x.grad), both):
        within(lp, want[0], e_logp.nan_to_num(0.0))
        within(h, want[1], e_h.nan_to_num(0.0))
        within(grad, want[4], e_grad.nan_to_num(0.0) + 4 * u * want[4].abs())


@pytest.mark.parametrize("vocab", [40, 3000, 8192, 20_000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite(device, vocab, dtype):
    """Among the legal logits they make the row NaN; its alternatives are those of the others."""
    z = randn(gen(vocab), 4, vocab, dtype=dtype)
    z[1, 3], z[2, vocab - 1], z[3] = float("nan"), math.inf, float("nan")
    bits = {torch.float32: torch.int32}.get(dtype, torch.int16)
    # (a NaN that signals, too)
    z.view(bits)[1, 5] = {torch.float32: 0x7F800001, torch.bfloat16: 0x7F81, torch.float16: 0x7C01}[dtype]
    tokens = torch.tensor([0, 1, 2, 3])
    want = net_ref.token_logprobs(z, tokens, None, 4)
    dev = z.to(device)
    logp, entropy, top_logp, top_tokens = (t.cpu() for t in net_ops.token_logprobs(
        dev, tokens.to(device), top=4))
    assert torch.equal(top_tokens, want[3])
    assert bool(torch.isfinite(logp[0])) and bool(torch.isnan(logp[1:]).all())
    assert bool(torch.isfinite(entropy[0])) and bool(torch.isnan(entropy[1:]).all())
    assert bool(torch.isnan(top_logp[1:3]).all()) and bool((top_logp[3] == -math.inf).all())
    zero = torch.zeros(4, device=device)
    grad = net_ops.token_logprobs_with_grad(dev, tokens.to(device), zero, None)[2]
    assert not bool(grad.any())  # (padding: no weight)


def test_near_certain_rows_keep_their_gradient(device):
    """1 - p of the given token has its bits where p rounds to 1."""
    for vocab in (64, 3000, 20_000):
        z = torch.full((1, vocab), -20.0)
        z[0, 7] = 0.0
        a = torch.ones(1)
        want = net_ref.token_logprobs(z, torch.tensor([7]), None, 0, a)[4]
        grad = net_ops.token_logprobs_with_grad(z.to(device), torch.tensor([7], device=device),
                                                a.to(device))[2]
        assert float(grad[0, 7]) == pytest.approx(float(want[0, 7]), rel=1e-4)


def test_repeats_graph_and_stream(device):
    z, tokens, legal, a, b = (t.to(device) for t in rows_of(5, 40, 4672, torch.bfloat16, True))

    def step():
        return (*net_ops.token_logprobs(z, tokens, legal, 8),
                *net_ops.token_logprobs_with_grad(z, tokens, a, b, legal))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want))


def test_no_rows(device):
    z = torch.ones(0, 10, device=device)
    t = torch.zeros(0, dtype=torch.int32, device=device)
    out = net_ops.token_logprobs(z, t, top=3)
    assert [x.shape for x in out] == [(0,), (0,), (0, 3), (0, 3)]
    assert net_ops.token_logprobs_with_grad(z, t)[2].shape == (0, 10)


def test_offsets_past_32_bits(device):
    rows, vocab = 70, 2**26
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=device)
    z[-1, -5:] = 30.0
    tokens = torch.full((rows,), vocab - 1, device=device)
    logp, entropy, top_logp, top_tokens = net_ops.token_logprobs(z, tokens, top=5)
    assert top_tokens[-1].tolist() == list(range(vocab - 5, vocab))
    assert float(logp[0]) == pytest.approx(-math.log(vocab), rel=1e-4)
    want = -math.log(5 + (vocab - 5) * math.exp(-30.0))
    assert float(logp[-1]) == pytest.approx(want, rel=1e-4)
