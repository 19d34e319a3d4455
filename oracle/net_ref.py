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


# ---- norm and rotation of heads -------------------------------------------------------------
def _rotation(positions, frequencies, sections, dim, interleaved):
    """The rotation of each token as a matrix [tokens, dim, dim]."""
    pairs = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    r = torch.eye(dim, dtype=torch.float64).repeat(positions.shape[0], 1, 1)
    for j in range(pairs):
        t = positions[:, axis[j]].double() * frequencies[j]
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        r[:, a, a] = r[:, b, b] = torch.cos(t)
        r[:, a, b], r[:, b, a] = -torch.sin(t), torch.sin(t)
    return r


def head_norm_rotary(x, positions, frequencies, weight, eps, sections, interleaved):
    """One of q and k: x [tokens, heads, dim], positions [tokens, axes]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    r = _rotation(positions, frequencies, sections, x.shape[-1], interleaved)
    return torch.matmul(r[:, None], x[..., None])[..., 0]


def head_norm_rotary_grad(g, x, positions, frequencies, weight, eps, sections, interleaved):
    """(grad_x, grad_weight)."""
    r = _rotation(positions, frequencies, sections, x.shape[-1], interleaved)
    d = torch.matmul(r.transpose(1, 2)[:, None], g.double()[..., None])[..., 0]
    if weight is None:
        return d, None
    x, w = x.double(), weight.double()
    root = torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x / root
    dn = d * w
    return (dn - n * (dn * n).mean(-1, keepdim=True)) / root, (d * n).sum((0, 1))


# ---- attention ------------------------------------------------------------------------------
def attention(q, k, v, scale, causal, grad=None):
    """One sequence: q [queries, q_heads, dim], k and v [keys, k_heads, dim] (those in use).
    (out, lse), and with `grad` the gradients of q, k and v.  Hidden keys take no part, whatever
    they hold."""
    lq, heads, dim = q.shape
    lk, group = k.shape[0], heads // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(lq, heads, dim, dtype=torch.float64)
    lse = torch.full((lq, heads), -math.inf, dtype=torch.float64)
    back = [torch.zeros_like(t) for t in (q, k, v)]
    for h in range(heads):
        for i in range(lq):
            n = min(max(i + 1 + lk - lq, 0), lk) if causal else lk
            if n == 0:
                continue
            kk, vv = k[:n, h // group], v[:n, h // group]
            s = scale * (kk @ q[i, h])
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[i, h])
            out[i, h] = p @ vv
            if grad is not None:
                g = grad[i, h].double()
                dp = vv @ g
                ds = p * (dp - (p * dp).sum()) * scale
                back[0][i, h] = ds @ kk
                back[1][:n, h // group] += ds[:, None] * q[i, h]
                back[2][:n, h // group] += p[:, None] * g
    return (out, lse) if grad is None else (out, lse, *back)


# ---- log-probabilities of tokens ------------------------------------------------------------
def token_logprobs(logits, tokens, legal, top, a=None, b=None):
    """(logp, entropy, top_logp, top_tokens, gradient of sum(a logp + b entropy)), a row at a
    time."""
    rows, vocab = logits.shape
    logp, entropy = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    top_logp = torch.full((rows, top), -math.inf, dtype=torch.float64)
    top_tokens = torch.full((rows, top), -1, dtype=torch.int64)
    grad = torch.zeros(rows, vocab, dtype=torch.float64)
    for i in range(rows):
        z = logits[i].double()
        ok = legal[i].bool() if legal is not None else torch.ones(vocab, dtype=torch.bool)
        t = int(tokens[i])
        given = 0 <= t < vocab and bool(ok[t])
        if not bool((z[ok] != -math.inf).any()):  # (a NaN is not)
            continue
        zl = z.masked_fill(~ok, -math.inf)
        logq = torch.log_softmax(zl, 0)
        p = torch.exp(logq)
        plogp = torch.where(p == 0, 0.0, p * logq)
        entropy[i] = -plogp.sum()
        if given:
            logp[i] = logq[t]
        order = sorted((j for j in range(vocab) if bool(ok[j]) and float(z[j]) > -math.inf),
                       key=lambda j: (-float(z[j]), j))[:top] if top else []
        for j, at in enumerate(order):
            top_logp[i, j], top_tokens[i, j] = logq[at], at
        wl = float(a[i]) if a is not None and given else 0.0
        we = float(b[i]) if b is not None else 0.0
        if wl or we:
            g = -wl * p - we * torch.where(p == 0, 0.0, p * (logq + entropy[i]))
            if given:
                g[t] += wl
            grad[i] = torch.where(ok & (z != -math.inf), g, 0.0)
            if given:
                grad[i, t] = g[t]
    return logp, entropy, top_logp, top_tokens, grad
