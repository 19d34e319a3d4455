"""The operators of a policy network over board tokens and of its training on searches: what each
case does through ``omoknuni_quantum_amd.net_ops``, and the same operators in plain torch.

Four operators, each with the direction that training needs:

* the token embedding with a scale, and its gradient over the sorted tokens;
* the root-mean-square norm of a residual sum (with dropout on the branch in training), its output
  in 8 bits with scales for serving, and its gradients;
* dropout from a counter-based generator: the mask is formed again wherever it is needed;
* the clipped policy loss over legal actions with a KL term, either sampled at the action against
  a reference's log-probability or over the whole row against a search's policy, with its gradient.

A case is a dict of plain values with a "kind"; ``prepare`` makes its inputs from the seed on the
GPU, ``run`` is one pass.  ``own`` chooses between the plain forms and the package's operators.
"""
import functools
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
FP8_MAX = 448.0


# ---- cases ----------------------------------------------------------------------------------
def _embed(name, tokens, vocab, dim, dtype):
    return {"name": name, "kind": "embed", "tokens": tokens, "vocab": vocab, "dim": dim,
            "dtype": dtype}


def _embed_grad(name, tokens, vocab, dim, dtype, skew):
    return {"name": name, "kind": "embed_grad", "tokens": tokens, "vocab": vocab, "dim": dim,
            "dtype": dtype, "skew": skew}


def _norm(name, kind, rows, dim, dtype, p=0.0, group=0):
    c = {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype}
    c.update({"group": group} if kind == "norm_fp8" else {"p": p})
    return c


def _dropout(name, rows, dim, dtype, p):
    return {"name": name, "kind": "dropout", "rows": rows, "dim": dim, "dtype": dtype, "p": p}


def _loss(name, kind, rows, actions, dtype, kl, legal, stride=0):
    return {"name": name, "kind": kind, "rows": rows, "actions": actions, "dtype": dtype,
            "kl": kl, "legal": legal, "stride": max(stride, actions)}


def listed():
    return [
        # serving one Gomoku position: 225 cells, a row of the table for each cell and content
        _embed("embed_position", 225, 675, 128, "bfloat16"),
        # the table's gradient for a batch of 512 Gomoku positions
        _embed_grad("embed_grad_boards", 512 * 225, 675, 256, "bfloat16", 1.0),
        # the gradient of a large vocabulary's table, its tokens as unevenly used as in text
        _embed_grad("embed_grad_vocabulary", 131_071, 65_536, 1024, "bfloat16", 3.0),
        # serving one token: the 8-bit input of the next product, one scale for the row
        _norm("norm_fp8_token", "norm_fp8", 1, 4096, "bfloat16"),
        # serving the leaves of a wave: 32 Go positions, a scale for every 128 columns
        _norm("norm_fp8_wave", "norm_fp8", 32 * 361, 2048, "bfloat16", group=128),
        # training over a batch of 512 Gomoku positions: dropout, sum and norm of a narrow model
        _norm("norm_train_boards", "norm", 512 * 225, 256, "float16", p=0.1),
        # the gradients of the same step in a wide model
        _norm("norm_grad_wide", "norm_grad", 16_384, 4096, "bfloat16", p=0.1),
        # dropout of an odd activation in float32, and of a large one in bfloat16
        _dropout("dropout_odd", 1449, 361, "float32", 0.1),
        _dropout("dropout_large", 65_536, 4096, "bfloat16", 0.25),
        # the loss of a batch of 512 Gomoku positions against the search's policies
        _loss("loss_gomoku", "loss_grad", 512, 225, "float32", "target", True),
        # the loss over the chess move slots in evaluation: forward only, padded rows
        _loss("loss_chess", "loss", 4096, 4672, "bfloat16", "target", True, stride=4736),
        # the loss of a training step over a large vocabulary: every token is allowed
        _loss("loss_vocabulary", "loss_grad", 4096, 131_072, "bfloat16", "sampled", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: the most bytes that a drawn case of a kind has to move: no more than the largest listed one's
_MOST = {"embed": 500e6, "embed_grad": 400e6, "norm": 500e6, "norm_fp8": 500e6, "norm_grad": 500e6,
         "dropout": 1e9, "loss": 1e9, "loss_grad": 2e9}


def _draw(rng, kind):
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if kind in ("embed", "embed_grad"):
        board = rng.random() < 0.5
        cells = rng.randint(7, 19) ** 2
        tokens = cells * _log(rng, 1, 1024) if board else _log(rng, 1, 262_144)
        vocab = 3 * cells if board else _log(rng, 64, 131_072)
        dim = 8 * _log(rng, 4, 256) if rng.random() < 0.75 else _log(rng, 17, 2049)
        if kind == "embed":
            return _embed("", tokens, vocab, dim, dtype)
        return _embed_grad("", tokens, vocab, dim, dtype, 1.0 if board else rng.choice((1.0, 3.0)))
    if kind in ("norm", "norm_fp8", "norm_grad"):
        rows = _log(rng, 1, 200_000)
        dim = 64 * _log(rng, 1, 128) if rng.random() < 0.75 else _log(rng, 33, 8191)
        if kind == "norm_fp8":
            dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
            return _norm("", kind, rows, dim, dtype, group=rng.choice((0, 128)))
        return _norm("", kind, rows, dim, dtype, p=rng.choice((0.0, 0.1, 0.3)))
    if kind == "dropout":
        return _dropout("", _log(rng, 1, 262_144), _log(rng, 16, 8192), dtype,
                        rng.choice((0.1, 0.25, 0.5)))
    if rng.random() < 0.6:  # a game's actions
        actions = rng.choice((rng.randint(7, 19) ** 2, rng.randint(7, 19) ** 2 + 1, 4672))
        rows, legal = _log(rng, 1, 32_768), True
    else:
        actions = _log(rng, 1_000, 131_072)
        rows, legal = _log(rng, 1, 16_384), False
    kl = rng.choice(("none", "sampled", "target")) if actions <= 8192 else \
        rng.choice(("none", "sampled"))
    stride = actions if rng.random() < 0.5 else (actions + 63) // 64 * 64 + 64 * rng.randint(0, 2)
    return _loss("", kind, rows, actions, dtype, kl, legal, stride)


def draw(rng):
    kind = rng.choice(("embed", "embed_grad", "embed_grad", "norm", "norm_fp8", "norm_grad",
                       "dropout", "loss", "loss_grad", "loss_grad"))
    c = _draw(rng, kind)
    while work(c)["bytes"] > _MOST[kind]:
        c = _draw(rng, kind)
    return {k: v for k, v in c.items() if k != "name"}


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("embed", "embed_grad"):
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        if kind == "embed":
            return {"bytes": n * 4 + min(n, v) * d * e + n * d * e, "flops": n * d}
        return {"bytes": n * 4 + n * d * e + v * d * e, "flops": n * d + v * d}
    if kind.startswith("norm"):
        r, d = case["rows"], case["dim"]
        if kind == "norm":  # x, residual -> y, h
            return {"bytes": 4 * r * d * e + d * e, "flops": 6 * r * d}
        if kind == "norm_fp8":  # x, residual -> q, scales, h
            groups = -(-d // case["group"]) if case["group"] else 1
            return {"bytes": 3 * r * d * e + r * d + 4 * r * groups + d * e, "flops": 8 * r * d}
        # grad_y, grad_h, h -> grad_x, grad_residual (one tensor without dropout), grad_weight
        return {"bytes": (5 if case["p"] else 4) * r * d * e + 2 * d * e, "flops": 12 * r * d}
    if kind == "dropout":
        n = case["rows"] * case["dim"]
        return {"bytes": 2 * n * e, "flops": n}
    r, a = case["rows"], case["actions"]
    per = e * (2 if kind == "loss_grad" else 1)
    per += (1 if case["legal"] else 0) + (4 if case["kl"] == "target" else 0)
    return {"bytes": r * a * per + r * 40, "flops": (8 if kind == "loss_grad" else 4) * r * a}


# ---- inputs ---------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
    return x if scale == 1.0 else x.mul_(scale)


def _prepare_embed(c, g, dt):
    n, v, d = c["tokens"], c["vocab"], c["dim"]
    if c.get("skew", 1.0) == 1.0 and v % 3 == 0:
        # a board: row 3*cell + content; two cells in three are empty
        cells = v // 3
        content = torch.randint(0, 6, (n,), generator=g, device=DEVICE).sub_(3).clamp_(min=0)
        ids = (torch.arange(n, device=DEVICE) % cells) * 3 + content
    else:
        u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
        ids = (u.pow_(c.get("skew", 1.0)) * v).long().clamp_(max=v - 1)
    s = {"ids": ids.int(), "scale": math.sqrt(d)}
    if c["kind"] == "embed":
        s["weight"] = _randn(g, v, d, dtype=dt, scale=0.02)
    else:
        s["grad"] = _randn(g, n, d, dtype=dt, scale=0.01)
    return s


def _prepare_norm(c, g, dt):
    r, d = c["rows"], c["dim"]
    s = {"weight": torch.rand(d, generator=g, device=DEVICE).add_(0.5).to(dt)}
    if c["kind"] == "norm_grad":
        s["h"] = _randn(g, r, d, dtype=dt, scale=2.0)
        s["grad_y"], s["grad_h"] = _randn(g, r, d, dtype=dt), _randn(g, r, d, dtype=dt)
    else:
        s["x"], s["residual"] = _randn(g, r, d, dtype=dt), _randn(g, r, d, dtype=dt, scale=2.0)
    return s


def _prepare_loss(c, g, dt):
    r, a = c["rows"], c["actions"]
    wide = _randn(g, r, c["stride"], dtype=dt, scale=2.0)
    s = {"logits": wide[:, :a]}
    if c["legal"]:
        # from few legal actions (chess) to nearly all of them (an empty board); some rows are
        # over: nothing is legal there
        share = torch.rand(r, 1, generator=g, device=DEVICE) * (0.02 if a == 4672 else 0.9) + 0.01
        s["legal"] = torch.rand(r, a, generator=g, device=DEVICE) < share
        s["legal"][::17] = False
    lse, act = torch.empty(r, device=DEVICE), torch.empty(r, dtype=torch.int64, device=DEVICE)
    step = max(1, 2**28 // a)
    for i in range(0, r, step):
        z = s["logits"][i:i + step].float()
        if c["legal"]:
            z.masked_fill_(~s["legal"][i:i + step], -math.inf)
        lse[i:i + step] = torch.logsumexp(z, 1)
        # an action drawn from the policy itself: the largest logit plus Gumbel noise
        act[i:i + step] = z.sub_(torch.rand(z.shape, generator=g, device=DEVICE).clamp_(
            min=1e-9).log_().neg_().log_()).argmax(1)
    logp = s["logits"].gather(1, act[:, None])[:, 0].float() - lse
    logp = logp.nan_to_num(0.0, 0.0, 0.0)
    act[5::29] = -1  # padding
    s["actions"] = act.int()
    s["advantages"] = _randn(g, r)
    s["old_logp"] = logp + _randn(g, r, scale=0.3)
    s["row_weight"] = torch.full((r,), 1.0 / r, device=DEVICE)
    if c["kl"] == "sampled":
        s["ref_logp"] = logp + _randn(g, r, scale=0.5)
    if c["kl"] == "target":
        # visit counts of a search of 800 simulations, normalised
        p = _randn(g, r, a, scale=2.0)
        if c["legal"]:
            p.masked_fill_(~s["legal"], -math.inf)
        p = torch.softmax(p, 1).nan_to_num_(0.0).mul_(800).round_()
        s["target"] = p / p.sum(1, keepdim=True).clamp_(min=1.0)
    return s


def prepare(case, seed):
    g, dt, kind = _gen(seed), DTYPES[case["dtype"]], case["kind"]
    if kind in ("embed", "embed_grad"):
        s = _prepare_embed(case, g, dt)
    elif kind.startswith("norm"):
        s = _prepare_norm(case, g, dt)
    elif kind == "dropout":
        s = {"x": _randn(g, case["rows"], case["dim"], dtype=dt)}
    else:
        s = _prepare_loss(case, g, dt)
    s.update(case=dict(case), dtype=dt, seed=int(seed) * 7919 + 1, offset=int(seed) % 1000)
    return s


# ---- plain forms ----------------------------------------------------------------------------
def _i64(x):
    """A 64-bit word as the int64 of the same bits."""
    x &= (1 << 64) - 1
    return x - (1 << 64) if x >> 63 else x


_GOLDEN, _MUL1, _MUL2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB


def _mix(z):
    """SplitMix64's finaliser on int64 tensors (shifts are logical)."""
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * _i64(_MUL1)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * _i64(_MUL2)
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _mix_host(x):
    m = (1 << 64) - 1
    z = (x + _GOLDEN) & m
    z = ((z ^ (z >> 30)) * _MUL1) & m
    z = ((z ^ (z >> 27)) * _MUL2) & m
    return z ^ (z >> 31)


def _key(seed, offset):
    m = (1 << 64) - 1
    return _mix_host(_mix_host(seed & m) ^ (offset & m))


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _keep(rows, dim, p, seed, offset):
    """The mask of dropout: element (r, c) is kept where the 16 bits c % 4 of the word
    splitmix64(key + golden * (r * ceil(dim / 4) + c // 4)) are at least p * 65536."""
    quads = (dim + 3) // 4
    q = torch.arange(rows * quads, device=DEVICE, dtype=torch.int64)
    w = _mix(q * _i64(_GOLDEN) + _i64(_key(seed, offset) + _GOLDEN))
    bits = torch.stack((w, w >> 16, w >> 32, w >> 48), 1) & 0xFFFF
    return (bits >= _threshold(p)).view(rows, quads * 4)[:, :dim]


def _dropped(x, p, seed, offset):
    """x (float32, [rows, dim]) with its dropped elements zero and the others scaled."""
    t = _threshold(p)
    if t == 0:
        return x
    keep = _keep(x.shape[0], x.shape[1], p, seed, offset)
    return torch.where(keep, x * (65536.0 / max(65536 - t, 1)), torch.zeros_like(x))


def _plain_embed_grad(s):
    out = torch.zeros(s["case"]["vocab"], s["case"]["dim"], device=DEVICE)
    out.index_add_(0, s["ids"], s["grad"].float())
    return (out * s["scale"]).to(s["dtype"])


def _rms(h):
    return torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)


def _plain_norm(s):
    c = s["case"]
    h = s["residual"].float() + _dropped(s["x"].float(), c["p"], s["seed"], s["offset"])
    y = h * _rms(h) * s["weight"].float()
    return {"y": y.to(s["dtype"]), "h": h.to(s["dtype"])}


def _groups(y, group):
    """y as [rows, groups, columns of a group], the last group filled up with zeros."""
    r, d = y.shape
    group = group or d
    n = -(-d // group)
    y = torch.nn.functional.pad(y, (0, n * group - d)) if n * group != d else y
    return y.view(r, n, group)


def _plain_norm_fp8(s):
    h = s["residual"].float() + s["x"].float()
    y = h * _rms(h) * s["weight"].float()
    g = _groups(y, s["case"]["group"])
    scale = (g.abs().amax(2) / FP8_MAX).clamp(min=2.0**-126)
    q = (g / scale[:, :, None]).reshape(y.shape[0], -1)[:, :y.shape[1]]
    return {"q": q.to(torch.float8_e4m3fn), "scales": scale, "h": h.to(s["dtype"])}


def _plain_norm_grad(s):
    c = s["case"]
    h, gy, w = s["h"].float(), s["grad_y"].float(), s["weight"].float()
    inv = _rms(h)
    n = h * inv
    gw = gy * w
    dh = (gw - n * (gw * n).mean(1, keepdim=True)) * inv + s["grad_h"].float()
    dx = _dropped(dh, c["p"], s["seed"], s["offset"])
    return {"x": dx.to(s["dtype"]), "residual": dh.to(s["dtype"]),
            "weight": (gy * n).sum(0).to(s["dtype"])}


def _plain_loss(s, c, grad):
    lo, hi, beta = c["clip_low"], c["clip_high"], c["kl_coef"]
    z = s["logits"].float()
    a = z.shape[1]
    if "legal" in s:
        z = torch.where(s["legal"], z, torch.full_like(z, -math.inf))
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = e.sum(1, keepdim=True)
    live = (total != 0)[:, 0]
    lse = torch.where(live[:, None], m + torch.log(total), torch.zeros_like(m))
    act = s["actions"].long()
    at = act.clamp(0, a - 1)[:, None]
    taken = (act >= 0) & (act < a) & live
    if "legal" in s:
        taken = taken & s["legal"].gather(1, at)[:, 0]
    zero = torch.zeros_like(lse[:, 0])
    logp = torch.where(taken, (z.gather(1, at) - lse)[:, 0], zero)
    ratio = torch.exp(torch.where(taken, logp - s["old_logp"], zero))
    adv = s["advantages"]
    one, two = ratio * adv, torch.clamp(ratio, 1.0 - lo, 1.0 + hi) * adv
    loss = torch.where(taken, -torch.minimum(one, two), zero)
    d_logp = torch.where(taken & (one <= two), -one, zero)
    kl, mass, pi = zero, zero, None
    if "ref_logp" in s:
        d = s["ref_logp"] - logp
        kl = torch.where(taken, torch.expm1(d) - d, zero)
        d_logp = d_logp - torch.where(taken, beta * torch.expm1(d), zero)
    if "target" in s:
        pi = s["target"]
        use = (pi > 0) & live[:, None]
        use = use & s["legal"] if "legal" in s else use
        pi = torch.where(use, pi, torch.zeros_like(pi))
        term = pi * (torch.log(torch.where(use, pi, torch.ones_like(pi))) -
                     torch.where(use, z - lse, torch.zeros_like(z)))
        kl, mass = term.sum(1), pi.sum(1)
    loss = loss + beta * kl
    out = {"loss": loss, "logp": logp, "kl": kl}
    if grad:
        safe = torch.where(live[:, None], total, torch.ones_like(total))
        g = (e / safe) * (beta * mass - d_logp)[:, None]
        g.scatter_add_(1, at, d_logp[:, None])
        if pi is not None:
            g = g - beta * pi
        out["grad"] = (g * s["row_weight"][:, None]).to(s["dtype"])
    return out


CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.1


def _loss_args(c):
    return {"clip_low": CLIP_LOW, "clip_high": CLIP_HIGH,
            "kl_coef": 0.0 if c["kl"] == "none" else 1.0 if c["kl"] == "target" else KL_COEF}


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "embed":
        return (s["weight"].float()[s["ids"].long()] * s["scale"]).to(s["dtype"])
    if kind == "dropout":
        return _dropped(s["x"].float(), c["p"], s["seed"], s["offset"]).to(s["dtype"])
    if kind in ("loss", "loss_grad"):
        return _plain_loss(s, _loss_args(c), kind == "loss_grad")
    return {"embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_fp8": _plain_norm_fp8,
            "norm_grad": _plain_norm_grad}[kind](s)


# ---- the package's operators ----------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _ops():
    from omoknuni_quantum_amd import net_ops

    return net_ops


def _run_own(s):
    ops, c, kind = _ops(), s["case"], s["case"]["kind"]
    if kind == "embed":
        return ops.token_embedding(s["ids"], s["weight"], s["scale"])
    if kind == "embed_grad":
        return ops.token_embedding_grad(s["grad"], s["ids"], c["vocab"], s["scale"])
    if kind == "dropout":
        return ops.dropout(s["x"], c["p"], s["seed"], s["offset"])
    if kind == "norm":
        y, h = ops.add_rms_norm(s["x"], s["residual"], s["weight"], EPS, c["p"], s["seed"],
                                s["offset"])
        return {"y": y, "h": h}
    if kind == "norm_fp8":
        q, scales, h = ops.add_rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS, c["group"])
        return {"q": q, "scales": scales, "h": h}
    if kind == "norm_grad":
        gx, gr, gw = ops.add_rms_norm_grad(s["grad_y"], s["grad_h"], s["h"], s["weight"], EPS,
                                           c["p"], s["seed"], s["offset"])
        return {"x": gx, "residual": gr, "weight": gw}
    args = dict(_loss_args(c), ref_logp=s.get("ref_logp"), target=s.get("target"),
                legal=s.get("legal"))
    inputs = (s["logits"], s["actions"], s["advantages"], s["old_logp"])
    if kind == "loss":
        loss, logp, kl = ops.clipped_policy_loss(*inputs, **args)
        return {"loss": loss, "logp": logp, "kl": kl}
    loss, logp, kl, grad = ops.clipped_policy_loss_with_grad(*inputs, s["row_weight"], **args)
    return {"loss": loss, "logp": logp, "kl": kl, "grad": grad}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------
def _exact_keep(rows, dim, p, seed, offset):
    """The mask again, the 64-bit products from 32-bit halves and the bits one column at a time."""
    low = (1 << 32) - 1

    def times(hi, lo, k):
        kh, kl = k >> 32, k & low
        # lo*kl needs all 64 bits: split lo once more so that no product passes 63 bits
        a, b = (lo & 0xFFFF) * kl, (lo >> 16) * kl
        s = (a >> 16) + b
        carry, out = s >> 16, ((s & 0xFFFF) << 16) | (a & 0xFFFF)

        def wrap(x, y):
            return ((((x >> 16) * y & 0xFFFF) << 16) + (x & 0xFFFF) * y) & low

        return (carry + wrap(hi, kl) + wrap(lo, kh)) & low, out

    def shift_xor(hi, lo, n):
        return hi ^ (hi >> n), lo ^ (((hi << (32 - n)) | (lo >> n)) & low)

    quads = -(-dim // 4)
    start = (_key(seed, offset) + _GOLDEN) & ((1 << 64) - 1)
    q = torch.arange(rows * quads, device=DEVICE, dtype=torch.int64)
    hi, lo = times(q >> 32, q & low, _GOLDEN)
    lo = lo + (start & low)
    hi = (hi + (start >> 32) + (lo >> 32)) & low
    lo = lo & low
    hi, lo = times(*shift_xor(hi, lo, 30), _MUL1)
    hi, lo = times(*shift_xor(hi, lo, 27), _MUL2)
    hi, lo = shift_xor(hi, lo, 31)
    keep = torch.empty(rows, quads, 4, dtype=torch.bool, device=DEVICE)
    for j, part in enumerate((lo & 0xFFFF, lo >> 16, hi & 0xFFFF, hi >> 16)):
        keep[:, :, j] = (part >= _threshold(p)).view(rows, quads)
    return keep.reshape(rows, quads * 4)[:, :dim]


def _exact_dropped(x, p, seed, offset):
    t = _threshold(p)
    if not t:
        return x
    return torch.where(_exact_keep(*x.shape, p, seed, offset), x * 65536 / max(65536 - t, 1), 0.0)


def _exact_embed_grad(s, v, d):
    """Per vocabulary row, the difference of two prefix sums over the tokens in sorted order."""
    ids, order = torch.sort(s["ids"].long(), stable=True)
    ends = torch.searchsorted(ids, torch.arange(v, device=DEVICE), right=True)
    out = torch.empty(v, d, dtype=torch.float64, device=DEVICE)
    for j in range(0, d, 128):
        total = torch.cumsum(s["grad"][order, j:j + 128].double(), 0)
        total = torch.cat((torch.zeros_like(total[:1]), total))[ends]
        out[:, j:j + 128] = torch.diff(total, dim=0, prepend=torch.zeros_like(total[:1]))
    return out * s["scale"]


def _exact_norm(s, c):
    x, r, w = s["x"].double(), s["residual"].double(), s["weight"].double()
    h = r + _exact_dropped(x, c.get("p", 0.0), s["seed"], s["offset"])
    y = w * h / torch.sqrt((h * h).sum(1, keepdim=True) / c["dim"] + EPS)
    return y, h


def _exact_norm_fp8(s, c):
    y, h = _exact_norm(s, c)
    group = c["group"] or c["dim"]
    scales, values = [], []
    for j in range(0, c["dim"], group):
        part = y[:, j:j + group]
        scales.append(torch.clamp(part.abs().max(1)[0] / FP8_MAX, min=2.0**-126))
        values.append(part / scales[-1][:, None])
    return {"q": torch.cat(values, 1), "scales": torch.stack(scales, 1), "h": h}


def _exact_norm_grad(s, c):
    h, gy, w = s["h"].double(), s["grad_y"].double(), s["weight"].double()
    ms = (h * h).sum(1, keepdim=True) / c["dim"] + EPS
    dot = (gy * w * h).sum(1, keepdim=True) / c["dim"]
    dh = s["grad_h"].double() + gy * w / ms.sqrt() - h * dot / (ms * ms.sqrt())
    return {"x": _exact_dropped(dh, c["p"], s["seed"], s["offset"]), "residual": dh,
            "weight": (gy * h / ms.sqrt()).sum(0)}


def _exact_loss_rows(s, c, a, i, j):
    z = s["logits"][i:j].double()
    n = z.shape[0]
    allowed = s["legal"][i:j] if "legal" in s else torch.ones_like(z, dtype=torch.bool)
    logq = torch.log_softmax(z.masked_fill(~allowed, -math.inf), 1)
    live = allowed.any(1)
    act = s["actions"][i:j].long()
    rows = torch.arange(n, device=DEVICE)
    ok = live & (act >= 0) & (act < a)
    at = torch.where(ok, act, 0)
    ok = ok & allowed[rows, at]
    logp = torch.where(ok, logq[rows, at], 0.0)
    adv, old = s["advantages"][i:j].double(), s["old_logp"][i:j].double()
    ratio = torch.exp(logp - old)
    inside = torch.where(adv >= 0, ratio <= 1 + c["clip_high"], ratio >= 1 - c["clip_low"])
    bound = torch.where(adv >= 0, 1 + c["clip_high"], 1 - c["clip_low"])
    loss = torch.where(ok, -adv * torch.where(inside, ratio, bound), 0.0)
    slope = torch.where(ok & inside, -adv * ratio, 0.0)
    kl, push = torch.zeros_like(loss), torch.zeros_like(z)
    prob = torch.where(allowed & live[:, None], logq.exp(), 0.0)
    if "ref_logp" in s:
        x = torch.exp(s["ref_logp"][i:j].double() - logp)
        kl = torch.where(ok, x - torch.log(x) - 1, 0.0)
        slope = slope + c["kl_coef"] * torch.where(ok, 1 - x, 0.0)
    if "target" in s:
        pi = torch.where(allowed, s["target"][i:j].double(), 0.0)
        kl = torch.where(pi > 0, pi * (pi.clamp(min=1e-300).log() - logq), 0.0).sum(1)
        push = c["kl_coef"] * (pi.sum(1, keepdim=True) * prob - pi)
    loss = loss + c["kl_coef"] * kl
    g = push - slope[:, None] * prob
    g[rows, at] += slope
    return loss, logp, kl, g * s["row_weight"][i:j].double()[:, None]


def _exact_loss(s, case):
    c, a, r = _loss_args(case), case["actions"], case["rows"]
    step = max(1, 2**26 // a)
    parts = [_exact_loss_rows(s, c, a, i, min(r, i + step)) for i in range(0, r, step)]
    out = dict(zip(("loss", "logp", "kl", "grad"), (torch.cat(p) for p in zip(*parts))))
    if case["kind"] == "loss":
        del out["grad"]
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "embed":
        return torch.index_select(s["weight"], 0, s["ids"].long()).double() * s["scale"]
    if kind == "embed_grad":
        return _exact_embed_grad(s, case["vocab"], case["dim"])
    if kind == "norm":
        return dict(zip(("y", "h"), _exact_norm(s, case)))
    if kind == "norm_fp8":
        return _exact_norm_fp8(s, case)
    if kind == "norm_grad":
        return _exact_norm_grad(s, case)
    if kind == "dropout":
        return _exact_dropped(s["x"].double(), case["p"], s["seed"], s["offset"])
    return _exact_loss(s, case)
