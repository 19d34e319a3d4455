"""The policy network's operators in 64 bits on the host, from their definitions: what the tests
of omoknuni_quantum_amd.net_ops compare with.  Inputs are torch tensors of any type on the CPU;
results are float64."""
from __future__ import annotations

import math

import torch

M64 = (1 << 64) - 1
GOLDEN = 0x9E3779B97F4A7C15


def splitmix64(x: int) -> int:
    z = (x + GOLDEN) & M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M64
    return z ^ (z >> 31)


def threshold(p: float) -> int:
    return int(math.floor(p * 65536.0 + 0.5))


def keep_mask(rows: int, dim: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """bool [rows, dim], one Python integer at a time."""
    key, quads, t = splitmix64(splitmix64(seed & M64) ^ (offset & M64)), (dim + 3) // 4, threshold(p)
    out = torch.empty(rows, dim, dtype=torch.bool)
    for r in range(rows):
        bits = []
        for q in range(quads):
            w = splitmix64((key + GOLDEN * (r * quads + q)) & M64)
            bits += [(w >> (16 * j)) & 0xFFFF >= t for j in range(4)]
        out[r] = torch.tensor(bits[:dim])
    return out


def dropout(x, p, seed, offset):
    x = x.double()
    t = threshold(p)
    if t == 0:
        return x
    rows = x.reshape(-1, x.shape[-1])
    keep = keep_mask(*rows.shape, p, seed, offset)
    scaled = rows * (65536.0 / (65536 - t)) if t < 65536 else torch.zeros_like(rows)
    return torch.where(keep, scaled, 0.0).reshape(x.shape)


def embedding(ids, weight, scale):
    ids, w = ids.long(), weight.double()
    ok = (ids >= 0) & (ids < w.shape[0])
    return torch.where(ok[..., None], w[torch.where(ok, ids, 0)] * scale, 0.0)


def embedding_grad(grad, ids, rows, scale):
    ids, g = ids.long().reshape(-1), grad.double().reshape(-1, grad.shape[-1])
    ok = (ids >= 0) & (ids < rows)
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    return out.index_add_(0, ids[ok], g[ok]) * scale


def add_rms_norm(x, residual, weight, eps, p=0.0, seed=0, offset=0):
    """(y, h, r): r the inverse root mean square."""
    h = dropout(x, p, seed, offset)
    if residual is not None:
        h = h + residual.double()
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * r * weight.double(), h, r


def add_rms_norm_grad(grad_y, grad_h, h, weight, eps, p=0.0, seed=0, offset=0):
    """(grad_x, grad_residual, grad_weight)."""
    h, gy = h.double(), grad_y.double()
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n, g = h * r, gy * weight.double()
    d = r * (g - n * (g * n).mean(-1, keepdim=True))
    if grad_h is not None:
        d = d + grad_h.double()
    return dropout(d, p, seed, offset), d, (gy * n).reshape(-1, h.shape[-1]).sum(0)


def policy_loss(logits, actions, advantages, old_logp, clip_low, clip_high, kl_coef,
                ref_logp=None, target=None, legal=None):
    """A dict of loss, logp, kl, ratio and grad (of each row's own loss by its logits)."""
    z = logits.double()
    n, a = z.shape
    ok = legal if legal is not None else torch.ones(n, a, dtype=torch.bool)
    ok = ok.bool()
    live = (ok & (z != -math.inf)).any(1)  # (a NaN is not left out)
    z = torch.where(ok, z, -math.inf)
    # (about the largest logit, so that rows far from zero keep the bits of log-probabilities)
    top = torch.where(z.isnan(), -math.inf, z).amax(1, keepdim=True)
    z = z - torch.where(top.isfinite(), top, 0.0)
    lse = torch.where(live, torch.logsumexp(torch.where(live[:, None], z, 0.0), 1), 0.0)
    logq = torch.where(ok & live[:, None], z - lse[:, None], -math.inf)
    prob = torch.exp(logq)
    act = actions.long()
    inside = (act >= 0) & (act < a)
    at = torch.where(inside, act, 0)
    rows = torch.arange(n)
    taken = inside & live & ok[rows, at]
    logp = torch.where(taken, logq[rows, at], 0.0)
    adv = advantages.double()
    ratio = torch.where(taken, torch.exp(logp - old_logp.double()), 1.0)
    one = ratio * adv
    two = torch.clamp(ratio, 1.0 - clip_low, 1.0 + clip_high) * adv
    loss = torch.where(taken, -torch.minimum(one, two), 0.0)
    slope = torch.where(taken & (one <= two), -one, 0.0)
    kl, grad = torch.zeros(n, dtype=torch.float64), torch.zeros_like(z)
    if ref_logp is not None:
        d = ref_logp.double() - logp
        kl = torch.where(taken, torch.where(d == math.inf, d, torch.expm1(d) - d), 0.0)
        if kl_coef:
            slope = slope - torch.where(taken, kl_coef * torch.expm1(d), 0.0)
    if target is not None:
        pi = target.double()
        use = ok & live[:, None] & (pi > 0)
        pi = torch.where(use, pi, 0.0)
        log_pi = torch.log(torch.where(use, pi, 1.0))
        kl = torch.where(use, pi * (log_pi - torch.where(use, logq, 0.0)), 0.0).sum(1)
        grad = kl_coef * (pi.sum(1, keepdim=True) * prob - pi)
    if kl_coef:
        loss = loss + kl_coef * kl
    grad = grad - slope[:, None] * prob
    grad[rows, at] += torch.where(taken, slope, 0.0)
    grad = torch.where(ok, grad, 0.0)  # (whatever a row of NaN holds)
    return {"loss": loss, "logp": logp, "kl": kl, "ratio": ratio, "grad": grad, "taken": taken,
            "prob": prob, "slope": slope}
