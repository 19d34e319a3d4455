"""Attention on the GPU against its definition in 64 bits (oracle/net_ref.py), and its gradients.

Tolerances, u = 2^-24 and U the unit roundoff of the elements' type (2^-24, 2^-8, 2^-11).  A float32
sum of n products is within n u of the sum of their magnitudes, in any order; products of 16-bit
elements are exact.

* Scores: with A_ij = scale sum |q_id k_jd|, s_ij is off by at most (dim + 4) u A_ij.
* A probability before it is normalised, e^(s - m): relative E_p = 2 max_j (dim + 4) u A_ij (s and
  m) + 4 u (1 + max |s - m|) (the products with log2 e, the instruction of 2^x).
* out: sum_j p_ij |v_jd| times E_p for the numerator and as much for l, U for p's rounding to the
  type, and 2 (keys + 32) u for the two sums and the rescaling of a running maximum; float16 also
  2^-25 sum |v| where p is subnormal.  Then out's own rounding.
* lse: E_p + (keys + 32) u + 4 u |lse|.
* Gradients: p is formed again from s and the rounded lse: relative E_s = (dim + 4) u A + E_lse + 4 u
  (1 + |s| + |lse|).  dP_ij = g_i.v_j is off by dim u sum |g v|, delta_i by U sum |g out| (out is
  rounded) and what out is off by, times |g|, and dim u sum |g out|.  ds = p (dP - delta) scale is off
  by |ds| (E_s + 4 u) + p scale (the two), and by U |ds| for its rounding (subnormal float16:
  2^-25).  The sums over keys (rows) add (count + 32) u of their magnitudes; p is rounded for dv.
"""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_net_ops import DTYPES, TINY, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


def dense(q, k, v, scale, causal, grad):
    """The definition for one sequence as matrices, with the bounds above: dicts of values and
    bounds.  Hidden keys must be finite here."""
    dtype = q.dtype
    lq, heads, dim = q.shape
    lk, group = k.shape[0], heads // k.shape[1]
    rnd = 0.0 if dtype == torch.float32 else U[dtype]
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    Q, G = (t.double().transpose(0, 1) for t in (q, grad))
    K, V = (t.double().transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
    seen = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        seen = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + lk - lq
    s = scale * Q @ K.transpose(1, 2)
    a = scale * Q.abs() @ K.abs().transpose(1, 2) * (dim + 4) * u
    a = a.masked_fill(~seen, 0.0)
    z = s.masked_fill(~seen, -math.inf)
    live = seen.any(1)
    lse = torch.logsumexp(z, 2) if lk else torch.full((heads, lq), -math.inf).double()
    p = torch.where(seen & live[:, None], torch.exp(z - lse.clamp(min=-1e300)[..., None]), 0.0)
    spread = torch.where(seen, (z.amax(2, keepdim=True) - z), 0.0).amax(2) if lk else lse * 0
    spread = torch.where(live, spread, 0.0)
    e_p = (2 * a.amax(2) if lk else 0.0) + 4 * u * (1 + spread)
    out = p @ V
    b_out = (p @ V.abs()) * (2 * e_p + rnd + 2 * (lk + 32) * u)[..., None]
    b_out = b_out + tiny * (seen.double() @ V.abs())
    b_lse = e_p + (lk + 32) * u + 4 * u * lse.abs().nan_to_num(0.0, 0.0, 0.0)
    val = {"out": out, "lse": lse}
    bound = {"out": b_out, "lse": torch.where(live, b_lse, 0.0)}
    # gradients
    dp = G @ V.transpose(1, 2)
    delta = (G * out).sum(2, keepdim=True)
    ds = p * (dp - delta) * scale
    e_s = a + torch.where(live, b_lse, 0.0)[..., None] + \
        torch.where(seen, 4 * u * (1 + s.abs()), 0.0) + \
        4 * u * lse.abs().nan_to_num(0.0, 0.0, 0.0)[..., None]
    off = dim * u * (G.abs() @ V.abs().transpose(1, 2)) + \
        (G.abs() * ((U[dtype] + dim * u) * out.abs() + (1 + U[dtype]) * b_out)).sum(2, keepdim=True)
    b_ds = ds.abs() * (e_s + 4 * u) + p * scale * off * (1 + e_s)
    b_ds = b_ds + rnd * (ds.abs() + b_ds) + torch.where(seen, tiny, 0.0)
    b_pr = p * e_s + rnd * p * (1 + e_s) + torch.where(seen, tiny, 0.0)
    rows, keys = (group * lq + 32) * u, (lk + 32) * u

    def heads_of(t):  # sums over the heads of a group
        return t.view(heads // group, group, lk, dim).sum(1)

    val["q"] = ds @ K
    bound["q"] = b_ds @ K.abs() + keys * (ds.abs() @ K.abs())
    val["k"] = heads_of(ds.transpose(1, 2) @ Q)
    bound["k"] = heads_of(b_ds.transpose(1, 2) @ Q.abs() + rows * (ds.abs().transpose(1, 2) @ Q.abs()))
    val["v"] = heads_of(p.transpose(1, 2) @ G)
    bound["v"] = heads_of(b_pr.transpose(1, 2) @ G.abs() + rows * (p.transpose(1, 2) @ G.abs()))
    flat = {x: t.transpose(0, 1) for x, t in val.items()}
    return flat, {x: 1.01 * t.transpose(0, 1) for x, t in bound.items()}


def inputs(g, lq, lk, heads, kv_heads, dim, dtype):
    return (randn(g, lq, heads, dim, dtype=dtype, scale=2.0), randn(g, lk, kv_heads, dim, dtype=dtype),
            randn(g, lk, kv_heads, dim, dtype=dtype), randn(g, lq, heads, dim, dtype=dtype))


SHAPES = [  # lq, lk, heads, kv_heads, dim
    (1, 1, 1, 1, 8), (1, 200, 8, 2, 64), (3, 3, 2, 2, 1), (5, 5, 2, 1, 33), (64, 64, 2, 2, 32),
    (65, 130, 4, 2, 40), (225, 225, 2, 2, 32), (130, 40, 3, 1, 64), (33, 300, 4, 4, 100),
    (129, 257, 2, 1, 128), (40, 1000, 8, 1, 80), (7, 64, 5, 5, 17), (300, 129, 1, 1, 127),
]


def test_the_matrices_are_the_definition():
    g = gen(1)
    for lq, lk, causal in ((4, 6, False), (4, 6, True), (6, 3, True), (2, 0, True)):
        q, k, v, go = inputs(g, lq, lk, 4, 2, 5, torch.float32)
        want = net_ref.attention(q, k, v, 0.3, causal, go)
        got, _ = dense(q, k, v, 0.3, causal, go)
        for name, w in zip(("out", "lse", "q", "k", "v"), want):
            fine = torch.isfinite(w)
            assert torch.equal(fine, torch.isfinite(got[name])), name
            assert float((got[name] - w)[fine].abs().amax()) < 1e-12 if fine.any() else True, name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_batch(device, dtype, causal, shape):
    g = gen(hash(shape) % 1000)
    two = [inputs(g, *shape, dtype) for _ in range(2)]
    q, k, v, go = (torch.stack(t).to(device) for t in zip(*two))
    scale = shape[-1]**-0.5
    out, lse = net_ops.attention_with_lse(q, k, v, causal=causal)
    assert torch.equal(net_ops.attention(q, k, v, scale, causal), out)
    grads = net_ops.attention_grad(go, q, k, v, out, lse, causal=causal)
    for i, t in enumerate(two):
        want, bound = dense(*t[:3], scale, causal, t[3])
        for name, got in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
            within(got[i], want[name], bound[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 32), (3, 3, 50)])
def test_packed(device, dtype, causal, lengths, heads, kv_heads, dim):
    """Sequences of no rows, of one and of many, rows before the first and behind the last, and
    NaN in every row that no sequence uses."""
    g = gen(dim + 7 * causal)
    lq = [0, 1, 49, 0, 130, 7, 225, 64, 1, 0]
    lk = [3, 1, 49, 9, 140, 5, 225, 64, 300, 0]
    used = [min(n, max(0, n - 2 * i)) for i, n in enumerate(lk)] if lengths else lk
    lead, tail = 5, 9
    seqs = [inputs(g, a, b, heads, kv_heads, dim, dtype) for a, b in zip(lq, lk)]
    starts = [torch.tensor([lead] + n).cumsum(0) for n in (lq, lk)]
    nan = float("nan")

    def packed(i, counts):
        rest = seqs[0][i].shape[1:]
        parts = [torch.full((lead, *rest), nan, dtype=dtype)]
        for s, t in enumerate(seqs):
            t = t[i].clone()
            if i in (1, 2):
                t[used[s]:] = nan
            parts.append(t)
        return torch.cat(parts + [torch.full((tail, *rest), nan, dtype=dtype)]).to(device)

    q, k, v, go = (packed(i, n) for i, n in enumerate((lq, lk, lk, lq)))
    args = dict(causal=causal, q_starts=starts[0].int().to(device),
                k_starts=starts[1].int().to(device),
                k_lengths=torch.tensor(used, dtype=torch.int32, device=device) if lengths else None)
    out, lse = net_ops.attention_with_lse(q, k, v, **args)
    gq, gk, gv = net_ops.attention_grad(go, q, k, v, out, lse, **args)
    for t in (out, gq, gk, gv):  # rows of no sequence
        assert not bool(t[:lead].any()) and not bool(t[-tail:].any())
    assert bool((lse[:lead] == -math.inf).all()) and bool((lse[-tail:] == -math.inf).all())
    for s, (a, b, c, e) in enumerate(seqs):
        n = used[s]
        want, bound = dense(a, b[:n], c[:n], dim**-0.5, causal, e)
        rq = slice(int(starts[0][s]), int(starts[0][s]) + lq[s])
        k0 = int(starts[1][s])
        for name, got in (("out", out[rq]), ("lse", lse[rq]), ("q", gq[rq]),
                          ("k", gk[k0:k0 + n]), ("v", gv[k0:k0 + n])):
            within(got, want[name], bound[name])
        assert not bool(gk[k0 + n:k0 + lk[s]].any()) and not bool(gv[k0 + n:k0 + lk[s]].any())


def test_many_short_sequences(device):
    """More sequences than the search of starts takes at a time, of 0 to 3 rows."""
    g = gen(3)
    lens = torch.randint(0, 4, (5000,), generator=g)
    starts = torch.cat((torch.zeros(1, dtype=torch.long), lens.cumsum(0)))
    n = int(starts[-1])
    q, k, v, go = inputs(g, n, n, 2, 1, 16, torch.float32)
    s = starts.int().to(device)
    dev = [t.to(device) for t in (q, k, v, go)]
    out, lse = net_ops.attention_with_lse(*dev[:3], q_starts=s)
    grads = net_ops.attention_grad(dev[3], *dev[:3], out, lse, q_starts=s)
    got = [t.cpu() for t in (out, lse, *grads)]
    for i in list(range(0, 200)) + list(range(4800, 5000)):
        a, b = int(starts[i]), int(starts[i + 1])
        want, bound = dense(q[a:b], k[a:b], v[a:b], 0.25, False, go[a:b])
        for name, t in zip(("out", "lse", "q", "k", "v"), got):
            within(t[a:b], want[name], bound[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 2, 9])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 64), (4, 4, 128), (6, 2, 24)])
def test_cache(device, dtype, queries, heads, kv_heads, dim):
    """Few queries over caches that are partly filled; the rest of a cache is NaN."""
    g = gen(queries + dim)
    room, lens = 2100, [0, 1, 63, 64, 65, 700, 2099, 2100]
    seqs = [inputs(g, queries, room, heads, kv_heads, dim, dtype) for _ in lens]
    q, k, v, _ = (torch.stack(t) for t in zip(*seqs))
    for i, n in enumerate(lens):
        k[i, n:], v[i, n:] = float("nan"), float("nan")
    out, lse = net_ops.attention_with_lse(
        q.to(device), k.to(device), v.to(device), causal=True,
        k_lengths=torch.tensor(lens, dtype=torch.int32, device=device))
    for i, n in enumerate(lens):
        want, bound = dense(q[i], k[i, :n], v[i, :n], dim**-0.5, True, q[i])
        within(out[i], want["out"], bound["out"])
        within(lse[i], want["lse"], bound["lse"])


@pytest.mark.parametrize("bad", [float("nan"), math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_hidden_values_that_are_not_finite(device, dtype, bad):
    """In a causal sequence a query's row does not see what later keys hold, nor a key's gradient
    what earlier queries hold."""
    g, n = gen(9), 150
    q, k, v, go = inputs(g, n, n, 2, 1, 48, dtype)
    clean, b_clean = dense(q, k, v, 48**-0.5, True, go)
    at = 101
    kb, vb = k.clone(), v.clone()
    kb[at, 0, 3], vb[at, 0, 5] = bad, bad
    vb[at + 20, 0, 7] = bad
    dev = [t.to(device) for t in (q, kb, vb, go)]
    dev = [t[None] for t in dev]
    out, lse = net_ops.attention_with_lse(*dev[:3], causal=True)
    gq = net_ops.attention_grad(dev[3], *dev[:3], out, lse, causal=True)[0]
    for name, t in (("out", out), ("lse", lse), ("q", gq)):
        within(t[0, :at], clean[name][:at], b_clean[name][:at])
    # queries: rows before a key's own do not reach its gradients
    qb, gb = q.clone(), go.clone()
    qb[at, 0, 3], gb[at, 1, 5] = bad, bad
    dev = [t.to(device)[None] for t in (qb, k, v, gb)]
    out, lse = net_ops.attention_with_lse(*dev[:3], causal=True)
    _, gk, gv = net_ops.attention_grad(dev[3], *dev[:3], out, lse, causal=True)
    for name, t in (("k", gk), ("v", gv)):
        within(t[0, at + 1:], clean[name][at + 1:], b_clean[name][at + 1:])
        if bad != bad:
            assert bool(torch.isnan(t[0, :at + 1]).all())


def test_a_visible_infinity_comes_through(device):
    v = torch.ones(1, 70, 1, 16, device=device)
    v[0, 10, 0, 2], v[0, 69, 0, 3], v[0, 5, 0, 4] = math.inf, -math.inf, float("nan")
    q = torch.zeros(1, 70, 1, 16, device=device)
    out = net_ops.attention(q, q, v, causal=True).cpu()[0, :, 0]

    def ones(t):  # n times the rounded 1 / n, rounded: two roundings of u
        return bool(((t - 1).abs() <= 2 * u).all())

    assert ones(out[:10, 2]) and bool((out[10:, 2] == math.inf).all())
    assert ones(out[:69, 3]) and float(out[69, 3]) == -math.inf
    assert ones(out[:5, 4]) and bool(torch.isnan(out[5:, 4]).all())


def test_strides(device):
    """Slices of one product's output, heads before tokens, one key and value for a whole batch."""
    g = gen(4)
    h, hk, d, n = 4, 2, 24, 70
    qkv = randn(g, 3, n, h + 2 * hk, d, dtype=torch.bfloat16).to(device)
    q, k, v = qkv.split((h, hk, hk), 2)
    want = net_ops.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(net_ops.attention(q, k, v), want)
    swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(net_ops.attention(*swapped), want)
    shared = [t[:1].expand(3, -1, -1, -1) for t in (k, v)]
    assert torch.equal(net_ops.attention(q, *shared),
                       net_ops.attention(q, *(t.contiguous() for t in shared)))
    out, lse = net_ops.attention_with_lse(q, k, v)
    go = torch.ones_like(out)
    one = net_ops.attention_grad(go, q, k, v, out, lse)
    two = net_ops.attention_grad(go, q.contiguous(), k.contiguous(), v.contiguous(), out, lse)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_starts_out_of_range_are_cut(device):
    """Nothing outside the arrays is read or written; the rows in range are attended to."""
    g = gen(6)
    q, k, v, go = (t.to(device) for t in inputs(g, 40, 40, 2, 2, 32, torch.float32))
    starts = torch.tensor([0, 10, 1000], dtype=torch.int32, device=device)
    lengths = torch.tensor([99, -5], dtype=torch.int32, device=device)
    out, lse = net_ops.attention_with_lse(q, k, v, q_starts=starts, k_lengths=lengths)
    want = net_ops.attention(q[None, :10], k[None, :10], v[None, :10])
    assert torch.equal(out[:10], want[0])
    assert not bool(out[10:].any()) and bool((lse[10:] == -math.inf).all())
    grads = net_ops.attention_grad(go, q, k, v, out, lse, q_starts=starts, k_lengths=lengths)
    assert all(not bool(t[10:].any()) and bool(torch.isfinite(t).all()) for t in grads)


def test_empty(device):
    for lq, lk in ((0, 5), (5, 0), (0, 0)):
        q, k = torch.ones(2, lq, 2, 8, device=device), torch.ones(2, lk, 2, 8, device=device)
        out, lse = net_ops.attention_with_lse(q, k, k, causal=True)
        assert out.shape == q.shape and not bool(out.any())
        assert bool((lse == -math.inf).all())
        grads = net_ops.attention_grad(out, q, k, k, out, lse, causal=True)
        assert [t.shape for t in grads] == [q.shape, k.shape, k.shape]
        assert all(not bool(t.any()) for t in grads)
    none = torch.ones(0, 5, 2, 8, device=device)
    assert net_ops.attention(none, none, none).shape == none.shape


def test_autograd_is_the_gradient_and_repeats(device):
    g = gen(8)
    q, k, v, go = (t[None].to(device) for t in inputs(g, 90, 90, 4, 2, 32, torch.float32))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = net_ops.attention(*leaves, causal=True)
    # (a gradient in another order of dimensions)
    out.backward(go.transpose(1, 2).contiguous().transpose(1, 2))
    one = [t.grad for t in leaves]
    o, lse = net_ops.attention_with_lse(q, k, v, causal=True)
    for _ in range(2):
        two = net_ops.attention_grad(go, q, k, v, o, lse, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_gradients_against_differences(device):
    """The change of the loss along random directions; float32 sums of about 1e3 terms of order 1,
    differenced over 2e-2: 1e3 * 2^-24 * few / 2e-2 and the step's third order."""
    g = gen(12)
    q, k, v, go = (t[None].to(device) for t in inputs(g, 30, 40, 4, 2, 16, torch.float32))
    out, lse = net_ops.attention_with_lse(q, k, v, 0.2, True)
    grads = net_ops.attention_grad(go, q, k, v, out, lse, 0.2, True)
    for i, t in enumerate((q, k, v)):
        d = randn(g, *t.shape).to(device)
        args = [q, k, v]

        def at(x):
            args[i] = t + x * d
            return float((net_ops.attention(*args, 0.2, True).double() * go).sum())

        slope = (at(1e-2) - at(-1e-2)) / 2e-2
        assert slope == pytest.approx(float((grads[i].double() * d).sum()), rel=2e-3, abs=2e-2)


def test_streams_and_graph(device):
    """On a side stream, and captured and replayed between eager calls that use the same
    workspaces' memory."""
    g = gen(14)
    q, k, v, go = (t[None].to(device) for t in inputs(g, 200, 200, 4, 2, 64, torch.bfloat16))

    def step(scale=0.125):
        out, lse = net_ops.attention_with_lse(q, k, v, scale, True)
        return (out, lse, *net_ops.attention_grad(go, q, k, v, out, lse, scale, True))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        if i == 2:
            q.mul_(0.5)
            want = step()
        for t in held:
            t.zero_()
        graph.replay()
        step(0.3)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_offsets_past_32_bits(device):
    """A cache of more than 2^32 elements; the last sequence's rows are behind them."""
    n, room, d = 9, 2**20, 128
    k = torch.zeros(n, room, 4, d, dtype=torch.bfloat16, device=device)
    g = gen(15)
    row = randn(g, 3, 4, d, dtype=torch.bfloat16)
    k[-1, 100:103] = row.to(device)
    q = randn(g, n, 1, 4, d, dtype=torch.bfloat16)
    lens = torch.full((n,), 103, dtype=torch.int32, device=device)
    out = net_ops.attention(q.to(device), k, k, k_lengths=lens)
    want, bound = dense(q[-1], k[-1, :103].cpu(), k[-1, :103].cpu(), d**-0.5, False, q[-1])
    within(out[-1], want["out"], bound["out"])
    assert not bool(out[:-1].any())
