"""Edges of the policy network's operators on the GPU against their definitions in 64 bits
(oracle/net_ref.py): infinities, rows without weight, large differences of log-probabilities.

Tolerances are derived as in test_gpu_net_ops.py: u = 2^-24, counts of operations times u times a
magnitude taken from the 64-bit reference, plus the rounding to the result's type."""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_net_ops import check_loss, gen, loss_inputs, randn, u, within

pytestmark = pytest.mark.gpu


def check_autograd(dev, args, want):
    """The gradient of the two operators, from the statistics that the loss left, against that of
    the one: finite, and the same but for the exponentials' roundings."""
    z = dev["z"].detach().clone().requires_grad_()
    loss, _, _ = net_ops.clipped_policy_loss(z, dev["act"], dev["adv"], dev["old"], **args)
    (loss * dev["weight"]).sum().backward()
    fused = net_ops.clipped_policy_loss_with_grad(dev["z"], dev["act"], dev["adv"], dev["old"],
                                                  dev["weight"], **args)[3]
    got, fused = z.grad.cpu().double(), fused.cpu().double()
    assert bool(got.isfinite().all()) and bool(fused.isfinite().all())
    # e^(z - m) in one exponential or in two: |z - m| below 40 in the logits that count, each
    # product with log2(e) off by u relative; the target's part of a sum that may cancel
    size = want["grad"].abs() * dev["weight"].cpu().double()[:, None]
    if dev.get("target") is not None:
        size = size + dev["target"].cpu().double() * args["kl_coef"]
    size = size + 2 * want["prob"] * (want["slope"].abs()[:, None] + args["kl_coef"])
    assert bool(((got - fused).abs() <= (4 * 40 + 4) * u * size + 2.0**-120).all())


# ---- waves of a row without weight ----------------------------------------------------------
@pytest.mark.parametrize("cols", [600, 1024, 4672, 8192, 16_384, 20_000, 80_000])
@pytest.mark.parametrize("level", [-100.0, -1000.0])
@pytest.mark.parametrize("kl", ["none", "sampled", "target"])
@pytest.mark.parametrize("masked", [False, True])
def test_columns_of_minus_infinity_below_far_logits(device, cols, level, kl, masked):
    """Logits that the caller masked with -inf, 512 columns and more of them, where the others are
    far below zero: those actions have probability and gradient 0, whatever the largest logit."""
    rows = 12
    d = loss_inputs(rows, cols, torch.float32, kl, False, cols)
    d["z"] = (d["z"] + level).float()
    away = torch.zeros(rows, cols, dtype=torch.bool)
    away[0::3, :512] = True
    away[1::3, 512:] = True
    away[2::3, 40:cols - 40] = True
    d["z"][away] = -math.inf
    if masked:
        d["legal"] = torch.rand(rows, cols, generator=gen(cols)) < 0.7
    open_ = ~away if not masked else ~away & d["legal"]
    for i in range(rows):  # an action that can be taken
        if 0 <= int(d["act"][i]) < cols:
            d["act"][i] = int(open_[i].nonzero()[i % 7])
    ref = net_ref.policy_loss(d["z"], d["act"], d["adv"], torch.zeros(rows), 0.2, 0.3, 0.0,
                              legal=d["legal"])
    d["old"] = (ref["logp"] + randn(gen(1), rows, scale=0.1)).float()
    if kl == "sampled":
        d["ref"] = (ref["logp"] + randn(gen(2), rows, scale=0.1)).float()
    if kl == "target":
        d["target"][away] = 0.0
    coef = {"none": 0.0, "sampled": 0.3, "target": 1.0}[kl]
    # (a bound relative to logits of 1000 over 800 terms decides nothing about the clipping)
    dev, args, want = check_loss(device, d, coef, with_grad=cols <= 16_384 or level > -500)
    assert bool(want["grad"].isfinite().all())
    check_autograd(dev, args, want)


# ---- the sampled kl's ends ------------------------------------------------------------------
def sampled_rows(cols, rows, seed):
    """Rows whose old log-probability is the present one: a ratio of 1, inside the clipping."""
    g = gen(seed)
    z = randn(g, rows, cols)
    act = torch.randint(0, cols, (rows,), generator=g)
    logp = net_ref.policy_loss(z, act, torch.zeros(rows), torch.zeros(rows), 0.2, 0.2,
                               0.0)["logp"]
    return z, act, torch.ones(rows), logp


def sampled(device, z, act, adv, old, ref, coef, dtype=torch.float32):
    args = dict(clip_low=0.2, clip_high=0.2, kl_coef=coef, ref_logp=ref.float().to(device))
    rest = act.to(device), adv.to(device), old.float().to(device)
    one = [t.cpu() for t in net_ops.clipped_policy_loss_with_grad(z.to(device), *rest, None,
                                                                  **args)]
    x = z.to(device).requires_grad_()
    two = net_ops.clipped_policy_loss(x, *rest, **args)
    two[0].backward(torch.ones_like(two[0]))
    two = [t.detach().cpu() for t in (*two, x.grad)]
    want = net_ref.policy_loss(z, act, adv, old.float(), 0.2, 0.2, coef, ref.float())
    return (one, two), want


def slope_bounds(want, act, coef, e_kl_slope):
    """Of the gradient, rounded to float32: the slope's error at the taken action and, times the
    probabilities, at the others, which have their own."""
    rows, cols = want["grad"].shape
    e_logp = 800 * u * (6.0 + math.log(cols))
    e_slope = 2 * e_logp + 4 * u + coef * e_kl_slope
    bound = want["prob"] * (want["slope"].abs() * 3 * e_logp + e_slope)[:, None]
    bound[torch.arange(rows), act] += e_slope
    return bound + 8 * u * want["grad"].abs()


@pytest.mark.parametrize("cols", [9, 300, 1024, 20_000, 80_000])
def test_sampled_kl_that_is_only_watched(device, cols):
    """No coefficient: a kl that overflows reaches neither the loss nor the gradient."""
    z, act, adv, logp = sampled_rows(cols, 6, cols)
    outs, want = sampled(device, z, act, adv, logp, logp + 100.0, 0.0)
    e_logp = 800 * u * (6.0 + math.log(cols))
    for out in outs:
        assert bool((out[2] == math.inf).all())
        within(out[0], want["loss"], 2 * e_logp + 4 * u)
        within(out[3], want["grad"], slope_bounds(want, act, 0.0, 0.0))


@pytest.mark.parametrize("cols", [9, 300, 1024, 20_000, 80_000])
@pytest.mark.parametrize("d", [-1000.0, -1e6, -math.inf])
def test_sampled_kl_far_below_the_action(device, cols, d):
    """The derivative of e^d - 1 - d is -1 to the last bit there."""
    z, act, adv, logp = sampled_rows(cols, 6, cols)
    outs, want = sampled(device, z, act, adv, logp, logp + d, 0.3)
    assert bool(want["grad"].isfinite().all())
    e_logp = 800 * u * (6.0 + math.log(cols))
    for out in outs:
        within(out[2], want["kl"], 4 * u * abs(d) + 2 * e_logp if d > -math.inf else 0.0)
        within(out[3], want["grad"], slope_bounds(want, act, 0.3, u))


@pytest.mark.parametrize("cols", [2, 300, 1024, 20_000, 80_000])
def test_sampled_kl_of_an_action_without_weight(device, cols):
    """A legal action of probability 0 was taken: the kl is infinite, as it is against a target."""
    z, act, adv, logp = sampled_rows(cols, 5, cols)
    z[torch.arange(5), act] = -math.inf
    for coef in (0.0, 0.3):
        outs, want = sampled(device, z, act, adv, logp, logp, coef)
        assert bool((want["kl"] == math.inf).all())
        for out in outs:
            assert bool((out[1] == -math.inf).all()) and bool((out[2] == math.inf).all())
            assert bool((out[0] == (math.inf if coef else 0.0)).all())
            if not coef:
                assert not bool(out[3].any())
    # a reference that is infinitely more likely, only watched
    z, act, adv, logp = sampled_rows(cols, 6, cols)
    outs, _ = sampled(device, z, act, adv, logp, logp + math.inf, 0.0)
    want = net_ref.policy_loss(z, act, adv, logp.float(), 0.2, 0.2, 0.0)
    for out in outs:
        assert bool((out[2] == math.inf).all())
        within(out[0], want["loss"], 2 * 800 * u * (6.0 + math.log(cols)) + 4 * u)
        within(out[3], want["grad"], slope_bounds(want, act, 0.0, 0.0))


# ---- padding --------------------------------------------------------------------------------
@pytest.mark.parametrize("cols", [300, 1024, 20_000, 80_000])
def test_padding_with_a_target_of_nothing(device, cols):
    """A row without an action whose target is zero adds nothing to the loss: its gradient is 0
    whatever its logits hold."""
    z = torch.full((3, cols), float("nan"))
    z[2] = 1.0
    f, act = torch.ones(3, device=device), torch.full((3,), -1, device=device)
    pi = torch.zeros(3, cols, device=device)
    pi[1] = -1.0
    one = net_ops.clipped_policy_loss_with_grad(z.to(device), act, f, f, kl_coef=1.0, target=pi)
    x = z.to(device).requires_grad_()
    two = net_ops.clipped_policy_loss(x, act, f, f, kl_coef=1.0, target=pi)
    two[0].sum().backward()
    for out in (one, (*two, x.grad)):
        assert all(not bool(t.any()) for t in out)


def test_sampled_kl_that_overflows_has_an_infinite_gradient(device):
    """e^100 and more is beyond float32: the gradient is -inf at the taken action and inf elsewhere."""
    for cols in (64, 300, 1024, 20_000, 80_000):
        z, act, adv, logp = sampled_rows(cols, 4, cols)
        outs, _ = sampled(device, 0.01 * z, act, adv, logp, logp + 115.0, 0.3)
        taken = torch.zeros(4, cols, dtype=torch.bool)
        taken[torch.arange(4), act] = True
        for out in outs:
            assert bool((out[0] == math.inf).all()) and bool((out[2] == math.inf).all())
            assert bool((out[3][taken] == -math.inf).all())
            assert bool((out[3][~taken] == math.inf).all())


# ---- a backward pass by hand ----------------------------------------------------------------
def test_logits_that_go_on_backwards_with_the_gradient(device):
    """logits.backward(grad) from rows that record gradients; the loss itself has no backward."""
    g = gen(31)
    x, w = randn(g, 20, 16).to(device), randn(g, 16, 225).to(device).requires_grad_()
    act, f = torch.randint(0, 225, (20,), generator=g).to(device), randn(g, 20).to(device)
    logits = x @ w
    loss, logp, kl, grad = net_ops.clipped_policy_loss_with_grad(logits, act, f, f)
    with pytest.raises(RuntimeError, match="not implemented"):
        loss.sum().backward(retain_graph=True)
    logits.backward(grad)
    with torch.no_grad():
        want = x.t() @ net_ops.clipped_policy_loss_with_grad(x @ w, act, f, f)[3]
    assert torch.equal(w.grad, want) and not w.grad.requires_grad


# ---- logits at the type's lowest value ------------------------------------------------------
@pytest.mark.parametrize("cols", [49, 600, 4672, 16_384, 20_000, 80_000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kl", ["none", "target"])
def test_logits_masked_with_the_lowest_value(device, cols, dtype, kl):
    """By the caller, in part of a row (those actions have probability 0) or in all of it (all
    have the same)."""
    rows = 12
    d = loss_inputs(rows, cols, dtype, kl, False, cols + 1)
    low = torch.finfo(dtype).min
    away = torch.rand(rows, cols, generator=gen(cols)) < 0.5
    away[0::4] = True
    away[1::4] = False
    away[1::4, :min(cols - 9, 512)] = True
    d["z"][away] = low
    inside = (d["act"] >= 0) & (d["act"] < cols)
    for i in range(rows):  # an action that can be taken
        if inside[i] and i % 4:
            d["act"][i] = int((~away[i]).nonzero()[i % 5])
    if kl == "target":
        d["target"][away & (torch.arange(rows) % 4 != 0)[:, None]] = 0.0
    top = torch.where(away.all(1), math.log(cols), 20.0 + math.log(cols))
    ref = net_ref.policy_loss(d["z"], d["act"], d["adv"], torch.zeros(rows), 0.2, 0.3, 0.0)
    d["old"] = (ref["logp"] + randn(gen(3), rows, scale=0.1)).float()
    dev = {k: v.to(device) for k, v in d.items() if v is not None}
    coef = 1.0 if kl == "target" else 0.0
    want = net_ref.policy_loss(d["z"], d["act"], d["adv"], d["old"], 0.2, 0.3, coef,
                               target=d.get("target"))
    args = dict(clip_low=0.2, clip_high=0.3, kl_coef=coef, target=dev.get("target"), legal=None)
    out = net_ops.clipped_policy_loss_with_grad(dev["z"], dev["act"], dev["adv"], dev["old"],
                                                dev["weight"], **args)
    # sums of at most 800 terms in a row, about the largest logit
    e_logp = 800 * u * (top + 1.0)
    within(out[1], want["logp"], e_logp)
    if kl == "target":
        within(out[2], want["kl"], 2 * e_logp * (1.0 + d["target"].double().sum(1)))
    x = dev["z"].clone().requires_grad_()
    two = net_ops.clipped_policy_loss(x, dev["act"], dev["adv"], dev["old"], **args)
    (two[0] * dev["weight"]).sum().backward()
    # rows clear of the clipping's bounds, where the gradient jumps
    e_ratio = want["ratio"] * (2 * e_logp + 4 * u)
    edge = torch.minimum((want["ratio"] - 0.8).abs(), (want["ratio"] - 1.3).abs())
    sure = edge > 2 * e_ratio + 1e-9
    assert float(sure.double().mean()) > 0.7
    e_slope = d["adv"].double().abs() * e_ratio
    bound = want["prob"] * ((want["slope"].abs() + coef) * 3 * e_logp + e_slope)[:, None]
    bound[torch.arange(rows), d["act"].clamp(0, cols - 1)] += e_slope
    if kl == "target":
        bound = bound + 4 * u * d["target"].double()
    w = d["weight"].double()[:, None]
    bound = w * (bound + 8 * u * want["grad"].abs())
    for grad in (out[3], x.grad):
        within(grad[sure.to(device)], (want["grad"] * w)[sure], bound[sure])
