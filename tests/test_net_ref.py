"""The 64-bit definitions behind the tests of the policy network's operators: their gradients
against central differences, and the dropout mask's statistics."""
import math

import pytest
import torch

from oracle import net_ref


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _difference(f, x, v, step=1e-5):
    """The derivative of the scalar f along v at x."""
    return float((f(x + step * v) - f(x - step * v)) / (2 * step))


def _along(grad, v):
    return float((grad * v).sum())


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("with_h", [False, True])
def test_norm_gradient_is_the_difference(p, with_h):
    g = _gen(1)
    x, res = torch.randn(5, 11, generator=g).double(), torch.randn(5, 11, generator=g).double()
    w = torch.rand(11, generator=g).double() + 0.5
    gy, gh = torch.randn(5, 11, generator=g).double(), torch.randn(5, 11, generator=g).double()

    def value(x, res, w):
        y, h, _ = net_ref.add_rms_norm(x, res, w, 1e-6, p, 7, 3)
        return (y * gy).sum() + ((h * gh).sum() if with_h else 0.0)

    h = net_ref.add_rms_norm(x, res, w, 1e-6, p, 7, 3)[1]
    gx, gr, gw = net_ref.add_rms_norm_grad(gy, gh if with_h else None, h, w, 1e-6, p, 7, 3)
    for k, (at, grad) in enumerate(((x, gx), (res, gr), (w, gw))):
        v = torch.randn(at.shape, generator=g).double()
        args = [x, res, w]

        def f(t):
            args[k] = t
            return value(*args)

        # central differences: an error of step^2 times the third derivative, all of order 1
        assert _difference(f, at, v) == pytest.approx(_along(grad, v), rel=1e-6, abs=1e-6)


@pytest.mark.parametrize("kl", ["none", "sampled", "target"])
@pytest.mark.parametrize("masked", [False, True])
def test_loss_gradient_is_the_difference(kl, masked):
    g = _gen(2)
    n, a = 12, 9
    z = torch.randn(n, a, generator=g).double()
    legal = torch.rand(n, a, generator=g) < 0.6 if masked else None
    if masked:
        legal[3] = False
    act = torch.randint(-1, a, (n,), generator=g)
    adv, weight = torch.randn(n, generator=g).double(), torch.rand(n, generator=g).double()
    old = torch.randn(n, generator=g).double() * 0.3 - 2.0
    args = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.7, legal=legal)
    if kl == "sampled":
        args["ref_logp"] = torch.randn(n, generator=g).double() * 0.3 - 2.0
    if kl == "target":
        args["target"] = torch.softmax(torch.randn(n, a, generator=g).double() * 2, 1)
    got = net_ref.policy_loss(z, act, adv, old, **args)
    v = torch.randn(n, a, generator=g).double()
    slope = _difference(lambda t: (net_ref.policy_loss(t, act, adv, old, **args)["loss"] *
                                   weight).sum(), z, v)
    assert slope == pytest.approx(_along(got["grad"] * weight[:, None], v), rel=1e-6, abs=1e-6)
    if masked:
        assert bool((got["grad"][~legal] == 0).all())
        assert got["loss"][3] == got["logp"][3] == got["kl"][3] == 0


def test_embedding_gradient_is_the_difference():
    g = _gen(3)
    ids = torch.tensor([[0, 3, 3], [7, -1, 2]])
    w, up = torch.randn(5, 4, generator=g).double(), torch.randn(2, 3, 4, generator=g).double()
    v = torch.randn(5, 4, generator=g).double()
    slope = _difference(lambda t: (net_ref.embedding(ids, t, 1.5) * up).sum(), w, v)
    grad = net_ref.embedding_grad(up, ids, 5, 1.5)
    assert slope == pytest.approx(_along(grad, v), rel=1e-8, abs=1e-8)


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_dropout_mask_statistics(p):
    rows, dim = 200, 101
    keep = net_ref.keep_mask(rows, dim, p, 123, 4).double()
    n = rows * dim
    # five standard deviations of a binomial count, and of the product of neighbours
    assert abs(float(keep.mean()) - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)
    c = keep - (1 - p)
    for pair in (c[:, 1:] * c[:, :-1], c[1:] * c[:-1], c[:, 4:] * c[:, :-4]):
        assert abs(float(pair.mean())) < 5 * p * (1 - p) / math.sqrt(pair.numel())
    other = net_ref.keep_mask(rows, dim, p, 123, 5).double() - (1 - p)
    assert abs(float((c * other).mean())) < 5 * p * (1 - p) / math.sqrt(n)


@pytest.mark.parametrize("coef", [0.0, 0.5])
def test_sampled_kl_of_an_action_without_weight_is_infinite(coef):
    """e^d - 1 - d at d = inf: a legal action of probability 0, as it is against a target."""
    z = torch.tensor([[-math.inf, 0.0, 1.0]])
    got = net_ref.policy_loss(z, torch.tensor([0]), torch.ones(1), torch.zeros(1), 0.2, 0.2, coef,
                              ref_logp=torch.tensor([-1.0]))
    assert float(got["logp"][0]) == -math.inf and float(got["kl"][0]) == math.inf
    assert float(got["loss"][0]) == (math.inf if coef else 0.0)
    if not coef:
        assert not bool(got["grad"].any())


def test_loss_definition_far_from_zero_and_of_nan():
    """Logits at the type's lowest value keep the bits of their log-probabilities, NaN among the
    legal logits reaches the results, and illegal actions have gradient 0 all the same."""
    low = torch.finfo(torch.float32).min
    z = torch.tensor([[low] * 4, [math.nan] * 4, [math.nan, 1.0, 2.0, 3.0]])
    legal = torch.tensor([[True] * 4, [True] * 3 + [False], [True, True, False, True]])
    f = torch.ones(3)
    got = net_ref.policy_loss(z, torch.tensor([2, 1, 1]), f, -math.log(4.0) * f, 0.2, 0.2, 0.0,
                              legal=legal)
    assert float(got["logp"][0]) == pytest.approx(-math.log(4.0), rel=1e-12)
    assert got["grad"][0].tolist() == pytest.approx([0.25, 0.25, -0.75, 0.25], rel=1e-6)
    for row in (1, 2):
        assert math.isnan(got["logp"][row]) and math.isnan(got["loss"][row])
        assert torch.equal(got["grad"][row].isnan(), legal[row])
        assert not bool(got["grad"][row][~legal[row]].any())
