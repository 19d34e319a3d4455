"""The operators of a policy network whose cells attend to one another, and of what such a policy
says of given moves: what each case does through ``omoknuni_quantum_amd.net_ops``, and the same
operators in plain torch.

Three operators, each with the direction that training needs:

* the norm of each head of queries and keys with the rotation by their positions along one or
  more axes (row and column of a cell), and its gradients;
* attention with grouped heads over a batch, over packed sequences of different lengths (boards of
  different sizes, prompts) and of few queries over a cache, and its gradients;
* the log-probabilities of given tokens over the legal ones, with the entropy and the best
  alternatives, and their gradient.

A case is a dict of plain values with a "kind"; ``prepare`` makes its inputs from the seed on the
GPU, ``run`` is one pass.  ``own`` chooses between the plain forms and the package's operators.
"""
import functools
import math
import random

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---- cases ----------------------------------------------------------------------------------
def _rotary(name, kind, tokens, heads, kv_heads, dim, dtype, axes=1, norm=True, turned=0,
            interleaved=False, far=0):
    """`turned`: the pairs that rotate (0: all); `far`: the first position."""
    return {"name": name, "kind": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "axes": axes, "norm": norm,
            "turned": turned or dim // 2, "interleaved": interleaved, "far": far}


def _attention(name, kind, layout, n, length, heads, kv_heads, dim, dtype, causal, queries=0,
               mix=0):
    """layout "equal": n sequences of `length`; "boards": n boards of 7 x 7 to 19 x 19 cells,
    packed; "texts": n packed sequences of 1 to `length` tokens; "cache": `queries` tokens each
    over n caches of `length` rows, of which 1 to all are filled."""
    return {"name": name, "kind": kind, "layout": layout, "n": n, "length": length,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal,
            "queries": queries, "mix": mix}


def _logprobs(name, kind, rows, vocab, dtype, legal, top=0, stride=0):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype,
            "legal": legal, "top": top, "stride": max(stride, vocab)}


def listed():
    return [
        # serving one token of a sequence far along, grouped heads
        _rotary("rotary_token", "rotary", 1, 32, 8, 128, "bfloat16", far=100_003),
        # training over a batch of 512 Gomoku positions: rows and columns as two axes
        _rotary("rotary_boards", "rotary", 512 * 225, 4, 4, 32, "float32", axes=2),
        # the gradients for a long batch of a wide model with three axes
        _rotary("rotary_grad_wide", "rotary_grad", 16_384, 32, 8, 128, "bfloat16", axes=3),
        # serving the leaves of a wave: 32 Gomoku positions
        _attention("attention_wave", "attention", "equal", 32, 225, 8, 8, 64, "bfloat16", False),
        # the same for a network of the package's default width, trained in float32
        _attention("attention_train_float", "attention_train", "equal", 64, 225, 4, 4, 32,
                   "float32", False),
        # training on boards of every size in one batch
        _attention("attention_train_boards", "attention_train", "boards", 256, 0, 8, 4, 64,
                   "float16", False, mix=1),
        # prompts of different lengths, packed
        _attention("attention_prompts", "attention", "texts", 8, 8192, 32, 8, 128, "bfloat16",
                   True, mix=2),
        # a training step over long sequences
        _attention("attention_train_long", "attention_train", "equal", 2, 4096, 16, 4, 128,
                   "bfloat16", True),
        # serving single tokens of 64 sequences over their caches
        _attention("attention_token", "attention", "cache", 64, 8192, 32, 8, 128, "bfloat16",
                   True, queries=1, mix=3),
        # what the policy says of the moves of 64 searched Gomoku positions, and its best five
        _logprobs("logprobs_moves", "logprobs", 64, 225, "float32", True, top=5),
        # the tokens of a batch under a large vocabulary, with their alternatives
        _logprobs("logprobs_vocabulary", "logprobs", 2048, 131_072, "bfloat16", False, top=8),
        # training with an entropy bonus over the chess move slots, padded rows
        _logprobs("logprobs_grad_chess", "logprobs_grad", 8192, 4672, "bfloat16", True,
                  stride=4736),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: the most that a drawn case of a kind has to move and compute: no more than the largest listed
_MOST = {"rotary": (230e6, 1e12), "rotary_grad": (500e6, 1e12), "attention": (2e9, 6e11),
         "attention_train": (1e9, 4e11), "logprobs": (530e6, 1e12), "logprobs_grad": (190e6, 1e12)}


def _draw(rng, kind):
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 8))
    if kind.startswith("rotary"):
        dim = 16 * rng.randint(1, 16) if rng.random() < 0.75 else rng.randint(9, 255)
        turned = dim // 2 if rng.random() < 0.7 else rng.randint(3, dim // 2)
        return _rotary("", kind, _log(rng, 1, 131_072), heads, kv, dim, dtype,
                       axes=rng.randint(1, 3), norm=rng.random() < 0.8, turned=turned,
                       interleaved=rng.random() < 0.3, far=rng.choice((0, 0, 5_000, 900_001)))
    if kind.startswith("attention"):
        dim = 16 * rng.randint(1, 8) if rng.random() < 0.75 else rng.randint(9, 127)
        layout = rng.choice(("equal", "boards", "texts") if kind == "attention_train" else
                            ("equal", "boards", "texts", "cache", "cache"))
        n = _log(rng, 1, 512)
        length = {"equal": rng.choice((rng.randint(7, 19)**2, _log(rng, 1, 8192))), "boards": 0,
                  "texts": _log(rng, 16, 8192), "cache": _log(rng, 16, 65_536)}[layout]
        causal = layout != "boards" and rng.random() < 0.6
        queries = rng.choice((1, 1, 1, rng.randint(2, 24))) if layout == "cache" else 0
        return _attention("", kind, layout, n, length, heads, kv, dim, dtype, causal, queries,
                          rng.randint(0, 999))
    if rng.random() < 0.6:  # a game's actions
        vocab = rng.choice((rng.randint(7, 19)**2, rng.randint(7, 19)**2 + 1, 4672))
        rows, legal = _log(rng, 1, 32_768), True
    else:
        vocab = _log(rng, 1_000, 131_072)
        rows, legal = _log(rng, 1, 8_192), False
    stride = vocab if rng.random() < 0.5 else (vocab + 63) // 64 * 64 + 64 * rng.randint(0, 2)
    top = 0 if kind == "logprobs_grad" else rng.choice((0, 1, 5, 8, 20))
    return _logprobs("", kind, rows, vocab, dtype, legal, top, stride)


def draw(rng):
    kind = rng.choice(("rotary", "rotary_grad", "attention", "attention", "attention",
                       "attention_train", "attention_train", "logprobs", "logprobs_grad"))
    while True:
        c = _draw(rng, kind)
        need = work(c)
        if need["bytes"] <= _MOST[kind][0] and need["flops"] <= _MOST[kind][1]:
            return {k: v for k, v in c.items() if k != "name"}


def _lengths(c):
    """(queries, keys in use) of each sequence, lists."""
    rng, n = random.Random(c["mix"]), c["n"]
    if c["layout"] == "equal":
        return [c["length"]] * n, [c["length"]] * n
    if c["layout"] == "cache":
        return [c["queries"]] * n, [rng.randint(1, c["length"]) for _ in range(n)]
    if c["layout"] == "boards":
        cells = [rng.randint(7, 19)**2 for _ in range(n)]
    else:
        cells = [_log(rng, 1, c["length"]) for _ in range(n - 1)] + [c["length"]]
    return cells, cells


def _pairs(c):
    """The visible (query, key) pairs of a head."""
    total = 0
    for lq, lk in zip(*_lengths(c)):
        if c["causal"]:  # the last query sees every key
            seen = min(lq, lk)
            total += seen * (lk - seen) + seen * (seen + 1) // 2
        else:
            total += lq * lk
    return total


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind.startswith("rotary"):
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": n * e * (3 if kind == "rotary_grad" else 2) + 4 * case["tokens"],
                "flops": n * (16 if kind == "rotary_grad" else 8)}
    if kind.startswith("attention"):
        lq, lk = _lengths(case)
        q = sum(lq) * case["heads"] * case["dim"] * e
        kv = sum(lk) * case["kv_heads"] * case["dim"] * e
        flops = _pairs(case) * case["heads"] * case["dim"]
        if kind == "attention":  # q, k, v -> out
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * flops}
        # q, k, v, grad -> out, and the gradients of q, k, v
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * flops}
    r, v = case["rows"], case["vocab"]
    per = e * (2 if kind == "logprobs_grad" else 1) + (1 if case["legal"] else 0)
    return {"bytes": r * v * per + r * (16 + 12 * case["top"]),
            "flops": (10 if kind == "logprobs_grad" else 5) * r * v}


# ---- inputs ---------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
    return x if scale == 1.0 else x.mul_(scale)


def _sections(c):
    """The rotated pairs of each axis."""
    n, a = c["turned"], c["axes"]
    return [n // a + (1 if i < n % a else 0) for i in range(a)]


def _prepare_rotary(c, g, dt):
    t, h, hk, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    qkv = _randn(g, t, h + 2 * hk, d, dtype=dt, scale=1.5)  # one product's output
    s = {"q": qkv[:, :h], "k": qkv[:, h:h + hk]}
    step = torch.arange(t, device=DEVICE)
    axes = [step] if c["axes"] == 1 else [step % 225 // 15, step % 15] if c["axes"] == 2 else \
        [step // 1024, step % 1024 // 32, step % 32]
    s["positions"] = (torch.stack(axes, 1) + c["far"]).int()
    # each axis has its own range of frequencies
    s["frequencies"] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                                  for n in _sections(c)]).to(DEVICE)
    if c["norm"]:
        s["q_weight"] = torch.rand(d, generator=g, device=DEVICE).add_(0.5).to(dt)
        s["k_weight"] = torch.rand(d, generator=g, device=DEVICE).add_(0.5).to(dt)
    if c["kind"] == "rotary_grad":
        s["grad_q"], s["grad_k"] = _randn(g, t, h, d, dtype=dt), _randn(g, t, hk, d, dtype=dt)
    return s


def _starts(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return starts


def _prepare_attention(c, g, dt):
    lq, lk = _lengths(c)
    h, hk, d, n = c["heads"], c["kv_heads"], c["dim"], c["n"]
    s = {"lq": lq, "lk": lk, "scale": 1.0 / math.sqrt(d)}
    if c["layout"] in ("equal", "cache"):
        rows, keys = (n, lq[0]), (n, c["length"])
    else:
        rows = keys = (sum(lq),)
        s["q_starts"] = torch.tensor(_starts(lq), dtype=torch.int32, device=DEVICE)
    if c["layout"] == "cache":
        s["k_lengths"] = torch.tensor(lk, dtype=torch.int32, device=DEVICE)
    # normed queries and keys: scores of some units, as trained heads have
    s["q"] = _randn(g, *rows, h, d, dtype=dt, scale=2.0)
    s["k"], s["v"] = _randn(g, *keys, hk, d, dtype=dt), _randn(g, *keys, hk, d, dtype=dt)
    if c["kind"] == "attention_train":
        s["grad"] = _randn(g, *rows, h, d, dtype=dt)
    return s


def _prepare_logprobs(c, g, dt):
    r, v = c["rows"], c["vocab"]
    s = {"logits": _randn(g, r, c["stride"], dtype=dt, scale=2.0)[:, :v]}
    tokens = torch.randint(0, v, (r,), generator=g, device=DEVICE)
    if c["legal"]:
        # from few legal moves to nearly all of them; some rows are over: nothing is legal there
        share = torch.rand(r, 1, generator=g, device=DEVICE) * (0.02 if v == 4672 else 0.9) + 0.01
        s["legal"] = torch.rand(r, v, generator=g, device=DEVICE) < share
        s["legal"].scatter_(1, tokens[:, None], True)  # (the move that was played)
        s["legal"][::17] = False
    tokens[5::29] = -1  # padding
    s["tokens"] = tokens.int()
    if c["kind"] == "logprobs_grad":
        s["logp_weight"] = _randn(g, r, scale=1.0 / r)
        s["entropy_weight"] = torch.full((r,), 0.01 / r, device=DEVICE)
    return s


def prepare(case, seed):
    g, dt, kind = _gen(seed), DTYPES[case["dtype"]], case["kind"]
    make = _prepare_rotary if kind.startswith("rotary") else \
        _prepare_attention if kind.startswith("attention") else _prepare_logprobs
    s = make(case, g, dt)
    s.update(case=dict(case), dtype=dt)
    return s


# ---- plain forms ----------------------------------------------------------------------------
def _angles(s):
    """(cos, sin) [tokens, 1, pairs] in float32, of angles in 64 bits."""
    axis = [a for a, n in enumerate(_sections(s["case"])) for _ in range(n)]
    at = s["positions"][:, axis].double() * s["frequencies"]
    return torch.cos(at).float()[:, None], torch.sin(at).float()[:, None]


def _split(x, c):
    """The two halves of the rotated pairs, and what does not rotate."""
    n = c["turned"]
    if c["interleaved"]:
        return x[..., 0:2 * n:2], x[..., 1:2 * n:2], x[..., 2 * n:]
    return x[..., :n], x[..., n:2 * n], x[..., 2 * n:]


def _join(a, b, rest, c):
    if c["interleaved"]:
        return torch.cat((torch.stack((a, b), -1).flatten(-2), rest), -1)
    return torch.cat((a, b, rest), -1)


def _turn(x, cos, sin, c):
    a, b, rest = _split(x, c)
    return _join(a * cos - b * sin, b * cos + a * sin, rest, c)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        if c["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s[name + "_weight"].float()
        out[name] = _turn(x, cos, sin, c).to(s["dtype"])
    return out


def _plain_rotary_grad(s):
    c = s["case"]
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        x, g = s[name].float(), _turn(s["grad_" + name].float(), cos, -sin, c)
        if c["norm"]:
            w = s[name + "_weight"].float()
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            out[name + "_weight"] = (g * x * r).sum((0, 1)).to(s["dtype"])
            g = g * w
            g = r * (g - x * (r * r * (g * x).mean(-1, keepdim=True)))
        out[name] = g.to(s["dtype"])
    return out


#: scores that the plain attention holds at a time
_SCORES = 2**29


def _sequence_chunks(s):
    """Ranges of sequences and the heads of keys to take at a time."""
    lq, lk = s["lq"], s["lk"]
    h, hk = s["case"]["heads"], s["case"]["kv_heads"]
    i = 0
    while i < len(lq):
        j, q, k = i, 0, 0
        while j < len(lq) and (j == i or (j + 1 - i) * max(q, lq[j]) * max(k, lk[j]) * h <= _SCORES):
            q, k, j = max(q, lq[j]), max(k, lk[j]), j + 1
        heads = hk
        while heads > 1 and (j - i) * q * k * (h // hk) * heads > _SCORES:
            heads -= 1
        yield i, j, q, k, heads
        i = j


def _rows(starts, lengths, longest):
    """The rows of sequences as [sequences, longest] indices, and which of them exist."""
    at = torch.arange(longest, device=DEVICE)
    n, first = (torch.tensor(x, device=DEVICE)[:, None] for x in (lengths, starts))
    return torch.where(at < n, first + at, 0), at < n


def _grouped(x, rows, live, groups):
    """[sequences * groups, heads of a group * rows, dim] in float32, zero where no row is."""
    x = torch.where(live[:, :, None, None], x[rows].float(), 0.0)
    n, t, h, d = x.shape
    x = x.view(n, t, groups, h // groups, d).permute(0, 2, 3, 1, 4)
    return x.reshape(n * groups, h // groups * t, d)


def _plain_attention(s, grad):
    c, d = s["case"], s["case"]["dim"]
    h, hk = c["heads"], c["kv_heads"]
    per = h // hk
    lq, lk = s["lq"], s["lk"]
    q_at = _starts(lq)
    k_at = [i * c["length"] for i in range(c["n"] + 1)] if c["layout"] == "cache" else _starts(lk)
    flat = {x: s[x].reshape(-1, *s[x].shape[-2:]) for x in ("q", "k", "v", "grad") if x in s}
    out = {"out": torch.zeros_like(flat["q"])}
    if grad:
        out.update({x: torch.zeros_like(flat[x]) for x in ("q", "k", "v")})
    for i, j, most_q, most_k, step in _sequence_chunks(s):
        qr, q_live = _rows(q_at[i:j], lq[i:j], most_q)
        kr, k_live = _rows(k_at[i:j], lk[i:j], most_k)
        seen = q_live[:, :, None] & k_live[:, None, :]
        if c["causal"]:
            shift = torch.tensor([b - a for a, b in zip(lq[i:j], lk[i:j])], device=DEVICE)
            seen &= (torch.arange(most_k, device=DEVICE)[None, None, :] <=
                     torch.arange(most_q, device=DEVICE)[None, :, None] + shift[:, None, None])
        for a in range(0, hk, step):
            b = min(hk, a + step)
            hq, hkv = slice(a * per, b * per), slice(a, b)
            q = _grouped(flat["q"][:, hq], qr, q_live, b - a)
            k, v = (_grouped(flat[x][:, hkv], kr, k_live, b - a) for x in ("k", "v"))
            mask = seen[:, None, None].expand(-1, b - a, per, -1, -1).reshape(-1, q.shape[1], most_k)
            z = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(s["scale"])
            z.masked_fill_(~mask, -math.inf)
            top = z.amax(2, keepdim=True)
            z = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
            total = z.sum(2, keepdim=True)
            p = z.div_(torch.where(total == 0, 1.0, total))
            o = torch.bmm(p, v)

            def back(x, live, rows, into, heads, count):
                x = x.view(j - i, b - a, count, -1, d).permute(0, 3, 1, 2, 4)
                x = x.reshape(j - i, -1, (b - a) * count, d)
                into[:, heads][rows[live]] = x[live].to(into.dtype)

            back(o, q_live, qr, out["out"], hq, per)
            if grad:
                g = _grouped(flat["grad"][:, hq], qr, q_live, b - a)
                dv = torch.bmm(p.transpose(1, 2).contiguous(), g)
                ds = torch.bmm(g, v.transpose(1, 2).contiguous())
                ds = ds.sub_((g * o).sum(2, keepdim=True)).mul_(p).mul_(s["scale"])
                back(torch.bmm(ds, k), q_live, qr, out["q"], hq, per)
                back(torch.bmm(ds.transpose(1, 2).contiguous(), q), k_live, kr, out["k"], hkv, 1)
                back(dv, k_live, kr, out["v"], hkv, 1)
    out = {x: t.view_as(s["q"] if x == "out" else s[x]) for x, t in out.items()}
    return out if grad else out["out"]


def _order(z):
    """int64 keys of the logits that fall with the value and then rise with the index: no two of
    a row are alike."""
    bits = z.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    return (bits << 32) - torch.arange(z.shape[1], device=DEVICE)


def _plain_logprobs_rows(s, c, i, j, grad):
    z = s["logits"][i:j].float()
    if "legal" in s:
        z = torch.where(s["legal"][i:j], z, -math.inf)
    top = z.amax(1, keepdim=True)
    live = top[:, 0] != -math.inf
    x = z - torch.where(live[:, None], top, 0.0)
    e = torch.exp(x)
    total = torch.where(live[:, None], e.sum(1, keepdim=True), 1.0)
    tokens = s["tokens"][i:j].long()
    at = tokens.clamp(0, c["vocab"] - 1)[:, None]
    ok = (tokens >= 0) & (tokens < c["vocab"]) & live
    if "legal" in s:
        ok = ok & s["legal"][i:j].gather(1, at)[:, 0]
    log_total = torch.log(total)
    out = {"logp": torch.where(ok, (x.gather(1, at) - log_total)[:, 0], 0.0)}
    xe = torch.where(e > 0, e * x, 0.0)
    out["entropy"] = torch.where(live, (log_total - xe.sum(1, keepdim=True) / total)[:, 0], 0.0)
    if c["top"]:
        k = min(c["top"], c["vocab"])
        index = torch.topk(_order(z + 0.0), k, dim=1)[1]
        values = z.gather(1, index)
        fine = values != -math.inf
        pad = (0, c["top"] - k)
        logq = torch.where(fine, x.gather(1, index) - log_total, -math.inf)
        out["top_logp"] = torch.nn.functional.pad(logq, pad, value=-math.inf)
        out["top_tokens"] = torch.nn.functional.pad(torch.where(fine, index, -1), pad, value=-1)
    if grad:
        p = e / total
        a, b = s["logp_weight"][i:j, None], s["entropy_weight"][i:j, None]
        a = torch.where(ok[:, None], a, 0.0)
        logq = torch.where(e > 0, x - log_total, 0.0)
        g = -p * (a + b * (logq + out["entropy"][:, None]))
        g = torch.where(live[:, None], g, 0.0)
        out["grad"] = g.scatter_add_(1, at, a).to(s["dtype"])
    return out


def _plain_logprobs(s, grad):
    c = s["case"]
    step = max(1, 2**27 // c["vocab"])
    parts = [_plain_logprobs_rows(s, c, i, min(c["rows"], i + step), grad)
             for i in range(0, c["rows"], step)]
    return {x: torch.cat([p[x] for p in parts]) for x in parts[0]}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind.startswith("rotary"):
        return _plain_rotary(s) if kind == "rotary" else _plain_rotary_grad(s)
    if kind.startswith("attention"):
        return _plain_attention(s, kind == "attention_train")
    return _plain_logprobs(s, kind == "logprobs_grad")


# ---- the package's operators ----------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _ops():
    from omoknuni_quantum_amd import net_ops

    return net_ops


def _run_own(s):
    ops, c, kind = _ops(), s["case"], s["case"]["kind"]
    if kind.startswith("rotary"):
        args = (s["positions"], s["frequencies"], s.get("q_weight"), s.get("k_weight"), EPS,
                _sections(c), c["interleaved"])
        if kind == "rotary":
            q, k = ops.head_norm_rotary(s["q"], s["k"], *args)
            return {"q": q, "k": k}
        gq, gk, gqw, gkw = ops.head_norm_rotary_grad(s["grad_q"], s["grad_k"], s["q"], s["k"],
                                                     *args)
        out = {"q": gq, "k": gk}
        return dict(out, q_weight=gqw, k_weight=gkw) if c["norm"] else out
    if kind.startswith("attention"):
        args = {"scale": s["scale"], "causal": c["causal"], "q_starts": s.get("q_starts"),
                "k_starts": s.get("q_starts"), "k_lengths": s.get("k_lengths")}
        if kind == "attention":
            return ops.attention(s["q"], s["k"], s["v"], **args)
        out, lse = ops.attention_with_lse(s["q"], s["k"], s["v"], **args)
        gq, gk, gv = ops.attention_grad(s["grad"], s["q"], s["k"], s["v"], out, lse, **args)
        return {"out": out, "q": gq, "k": gk, "v": gv}
    if kind == "logprobs":
        logp, entropy, top_logp, top_tokens = ops.token_logprobs(
            s["logits"], s["tokens"], legal=s.get("legal"), top=c["top"])
        out = {"logp": logp, "entropy": entropy}
        return dict(out, top_logp=top_logp, top_tokens=top_tokens) if c["top"] else out
    logp, entropy, grad = ops.token_logprobs_with_grad(
        s["logits"], s["tokens"], s["logp_weight"], s["entropy_weight"], legal=s.get("legal"))
    return {"logp": logp, "entropy": entropy, "grad": grad}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------
def _exact_rotary(s, c):
    """The rotation as a product of complex numbers; gradients by the conjugate."""
    t, n = c["tokens"], c["turned"]
    edges = _starts(_sections(c))
    angle = torch.empty(t, n, dtype=torch.float64, device=DEVICE)
    for a in range(c["axes"]):
        part = slice(edges[a], edges[a + 1])
        angle[:, part] = torch.outer(s["positions"][:, a].double(), s["frequencies"][part])
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if c["interleaved"]:
        one, two = torch.arange(0, 2 * n, 2, device=DEVICE), torch.arange(1, 2 * n, 2, device=DEVICE)
    else:
        one, two = torch.arange(n, device=DEVICE), torch.arange(n, 2 * n, device=DEVICE)
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        ms = (x * x).sum(-1, keepdim=True) / c["dim"] + EPS
        w = s[name + "_weight"].double() if c["norm"] else None
        back = c["kind"] == "rotary_grad"
        y = s["grad_" + name].double() if back else x / ms.sqrt() * w if c["norm"] else x.clone()
        z = torch.complex(y[..., one], y[..., two]) * (turn.conj() if back else turn)
        y[..., one], y[..., two] = z.real, z.imag
        if back and c["norm"]:
            out[name + "_weight"] = (y * x / ms.sqrt()).sum((0, 1))
            dot = (y * w * x).sum(-1, keepdim=True) / c["dim"]
            y = y * w / ms.sqrt() - x * dot / (ms * ms.sqrt())
        out[name] = y
    return out


def _exact_attention(s, c):
    """A sequence and a head at a time."""
    per, train = c["heads"] // c["kv_heads"], c["kind"] == "attention_train"
    lq, lk = s["lq"], s["lk"]
    flat = {x: s[x].reshape(-1, *s[x].shape[-2:]) for x in ("q", "k", "v", "grad") if x in s}
    out = {x: torch.zeros(flat[y].shape, dtype=torch.float64, device=DEVICE)
           for x, y in (("out", "q"), ("q", "q"), ("k", "k"), ("v", "v"))}
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(lq, lk)):
        if c["layout"] == "cache":
            k0 = i * c["length"]
        hidden = torch.ones(nq, nk, dtype=torch.bool, device=DEVICE).triu(nk - nq + 1)
        for h in range(c["heads"]):
            q = flat["q"][q0:q0 + nq, h].double()
            k, v = (flat[x][k0:k0 + nk, h // per].double() for x in ("k", "v"))
            z = q @ k.T * s["scale"]
            if c["causal"]:
                z.masked_fill_(hidden, -math.inf)
            p = torch.softmax(z, 1).nan_to_num_(0.0)
            out["out"][q0:q0 + nq, h] = p @ v
            if train:
                g = flat["grad"][q0:q0 + nq, h].double()
                dp = g @ v.T
                dz = p * (dp - (p * dp).sum(1, keepdim=True)) * s["scale"]
                out["q"][q0:q0 + nq, h] = dz @ k
                out["k"][k0:k0 + nk, h // per] += dz.T @ q
                out["v"][k0:k0 + nk, h // per] += p.T @ g
        q0, k0 = q0 + nq, k0 + nk
    if not train:
        return out["out"].view_as(s["q"])
    return {x: t.view_as(s["q"] if x == "out" else s[x]) for x, t in out.items()}


def _exact_logprobs(s, c):
    rows, v, top = c["rows"], c["vocab"], c["top"]
    parts = []
    step = max(1, 2**26 // v)
    for i in range(0, rows, step):
        z = s["logits"][i:i + step].double()
        n = z.shape[0]
        legal = s["legal"][i:i + step] if "legal" in s else torch.ones_like(z, dtype=torch.bool)
        logq = torch.log_softmax(z.masked_fill(~legal, -math.inf), 1)
        p = torch.where(legal & legal.any(1, keepdim=True), logq.exp(), 0.0)
        entropy = -torch.where(p > 0, p * logq, 0.0).sum(1)
        token = s["tokens"][i:i + step].long()
        row = torch.arange(n, device=DEVICE)
        ok = (token >= 0) & (token < v)
        at = torch.where(ok, token, 0)
        ok = ok & legal[row, at]
        part = {"logp": torch.where(ok, logq[row, at], 0.0), "entropy": entropy}
        if top:
            left = z.masked_fill(~legal, -math.inf)
            values = torch.full((n, top), -math.inf, dtype=torch.float64, device=DEVICE)
            tokens = torch.full((n, top), -1, device=DEVICE)
            ramp = torch.arange(v, device=DEVICE)
            for j in range(min(top, v)):  # the best one left, the first of its equals
                best = left.max(1, keepdim=True)[0]
                index = torch.where(left == best, ramp, v).min(1)[0]
                there = best[:, 0] != -math.inf
                tokens[there, j] = index[there]
                values[there, j] = logq[row, index][there]
                left[row, index] = -math.inf
            part.update(top_logp=values, top_tokens=tokens)
        if c["kind"] == "logprobs_grad":
            a = torch.where(ok, s["logp_weight"][i:i + step].double(), 0.0)
            b = s["entropy_weight"][i:i + step].double()
            g = -a[:, None] * p
            g -= b[:, None] * torch.where(p > 0, p * (logq + entropy[:, None]), 0.0)
            g[row, at] += a
            part["grad"] = g
        parts.append(part)
    return {x: torch.cat([part[x] for part in parts]) for x in parts[0]}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind.startswith("rotary"):
        return _exact_rotary(s, case)
    if kind.startswith("attention"):
        return _exact_attention(s, case)
    return _exact_logprobs(s, case)
