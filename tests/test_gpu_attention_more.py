"""More of the attention on the GPU: heads in groups that do not divide a tile, rows of few keys whose
gradients are exact but for one rounding, keys in parts, graphs side by side, and heads that start
anywhere.  Bounds as in test_gpu_attention.py."""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from tests.test_gpu_attention import dense, inputs
from tests.test_gpu_net_ops import DTYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 1, 64), (10, 2, 32), (6, 1, 128), (7, 1, 20),
                                                (48, 1, 64)])
@pytest.mark.parametrize("lq,lk", [(90, 90), (31, 200)])
def test_groups_that_do_not_divide_a_tile(device, dtype, heads, kv_heads, dim, lq, lk):
    q, k, v, go = inputs(gen(heads + lq), lq, lk, heads, kv_heads, dim, dtype)
    want, bound = dense(q, k, v, dim**-0.5, True, go)
    q, k, v, go = (t[None].to(device) for t in (q, k, v, go))
    out, lse = net_ops.attention_with_lse(q, k, v, causal=True)
    got = (out, lse, *net_ops.attention_grad(go, q, k, v, out, lse, causal=True))
    for name, t in zip(("out", "lse", "q", "k", "v"), got):
        within(t[0], want[name], bound[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,dim,causal", [(1, 16, False), (5, 64, True), (30, 128, True),
                                          (64, 32, False), (65, 64, True), (128, 128, True),
                                          (128, 48, False)])
def test_few_keys_have_gradients_of_one_rounding(device, dtype, n, dim, causal):
    """delta is the sum of p dP here, and ds has twice the type's bits: dq is off by its own rounding,
    by U^2 for ds (and 2^-25 of what is subnormal in float16's second part), and by float32's: with
    e = (dim + 4) u max A + e_lse + 4 u (1 + |s| + |lse|) of a probability, D_ij = dim u sum |g v| of
    dP and n + 64 roundings of sums, |ds| 3 e + p scale (D + sum p (D + |dP| 3 e + |delta| 3 e))."""
    q, k, v, go = inputs(gen(n + dim), n, n, 2, 2, dim, dtype)
    scale = dim**-0.5
    dev = [t[None].to(device) for t in (q, k, v, go)]
    out, lse = net_ops.attention_with_lse(*dev[:3], scale, causal)
    got = net_ops.attention_grad(dev[3], *dev[:3], out, lse, scale, causal)[0][0].cpu().double()
    Q, K, V, G = (t.double().transpose(0, 1) for t in (q, k, v, go))
    seen = torch.ones(n, n, dtype=torch.bool)
    if causal:
        seen = seen.tril()
    s = (scale * Q @ K.transpose(1, 2)).masked_fill(~seen, -math.inf)
    p, l = torch.softmax(s, 2), torch.logsumexp(s, 2, keepdim=True)
    dp = G @ V.transpose(1, 2)
    delta = (p * dp).sum(2, keepdim=True)
    ds = p * (dp - delta) * scale
    a = scale * (Q.abs() @ K.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(2, keepdim=True)
    big = s.masked_fill(~seen, 0.0).abs().amax(2, keepdim=True)
    e = 3 * (dim + 4) * u * a + (n + 64) * u + 12 * u * (1 + big + l.abs())
    d = dim * u * (G.abs() @ V.abs().transpose(1, 2))
    b = ds.abs() * 3 * e + p * scale * (
        d + (p * (d + (dp.abs() + delta.abs()) * (3 * e + (n + 64) * u))).sum(2, keepdim=True))
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    b = b + U[dtype]**2 * ds.abs() + torch.where(seen, tiny, 0.0)
    want = (ds @ K).transpose(0, 1)
    bound = (b @ K.abs() + (n + 64) * u * (ds.abs() @ K.abs())).transpose(0, 1)
    off = (got - want).abs()
    assert bool((off <= 1.01 * (bound + U[dtype] * (want.abs() + bound)) + tiny).all()), \
        float((off / (bound + U[dtype] * want.abs() + 1e-30)).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk,heads,dim", [(1, 1024, 2, 64), (1, 4097, 3, 128), (40, 2050, 2, 32),
                                             (200, 1500, 1, 100)])
def test_keys_in_parts(device, dtype, lq, lk, heads, dim):
    q, k, v, go = inputs(gen(lq + lk), lq, lk, heads, heads, dim, dtype)
    want, bound = dense(q, k, v, dim**-0.5, True, go)
    out, lse = net_ops.attention_with_lse(*(t[None].to(device) for t in (q, k, v)), causal=True)
    within(out[0], want["out"], bound["out"])
    within(lse[0], want["lse"], bound["lse"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_with_values_that_are_not_finite(device, dtype):
    """What a query sees comes through from any part, what it does not see from none."""
    n, lk, at = 5, 2000, 1300
    q, k, v, go = inputs(gen(3), n, lk, 2, 2, 64, dtype)
    want, bound = dense(q, k[:, :], v, 0.125, True, go)
    for bad in (math.nan, math.inf):
        kb, vb = k.clone(), v.clone()
        vb[lk - 2, 0, 5], kb[lk - 1, 1, 3] = bad, math.nan  # (the last query alone sees the last key)
        out, lse = net_ops.attention_with_lse(*(t[None].to(device) for t in (q, kb, vb)), 0.125, True)
        out = out[0].cpu()
        within(out[:n - 2], want["out"][:n - 2], bound["out"][:n - 2])
        rest = torch.arange(64) != 5
        within(out[:, 0, rest], want["out"][:, 0, rest], bound["out"][:, 0, rest])
        seen = out[n - 2:, 0, 5].float()
        assert bool((seen == bad).all()) if bad == bad else bool(seen.isnan().all())
        assert bool(out[n - 1, 1].isnan().all()) and bool(out[n - 2, 1].isfinite().all())
        vb = v.clone()
        vb[at, 1, 0] = bad  # (in a tile that no mask cuts, of a part in the middle)
        out = net_ops.attention(*(t[None].to(device) for t in (q, k, vb)), 0.125, True)[0].cpu()
        hit = out[:, 1, 0].float()
        assert bool((hit == bad).all()) if bad == bad else bool(hit.isnan().all())
        within(out[:, :, 1:], want["out"][:, :, 1:], bound["out"][:, :, 1:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 33, 130])
def test_values_that_are_not_finite_reach_the_few_rows_that_see_them(device, dtype, rows):
    """In the last tile of a short sequence, for out and all gradients; columns past the rows' count
    among them."""
    dim, keys = 64, rows + 20
    q, k, v, go = inputs(gen(rows), rows, keys, 1, 1, dim, dtype)
    kb, vb = k.clone(), v.clone()
    vb[keys - 1, 0, 60] = math.inf  # the last row alone sees it
    dev = [t[None].to(device) for t in (q, kb, vb, go)]
    out = net_ops.attention(*dev[:3], causal=True)[0, :, 0].cpu()
    assert float(out[-1, 60]) == math.inf and bool(out[:-1].isfinite().all())
    assert bool(out[-1, :60].isfinite().all())
    # a key of infinity: the gradient of the query that sees it, and no other, is NaN there
    kb[keys - 1, 0, 60] = math.nan
    dev = [t[None].to(device) for t in (q, kb, v, go)]
    out, lse = net_ops.attention_with_lse(*dev[:3], causal=True)
    gq = net_ops.attention_grad(dev[3], *dev[:3], out, lse, causal=True)[0][0, :, 0].cpu()
    assert bool(gq[-1].isnan().all()) and bool(gq[:-1].isfinite().all())
    # a gradient that is not finite reaches the keys that its row sees
    gb = go.clone()
    gb[0, 0, 60] = math.nan
    dev = [t[None].to(device) for t in (q, k, v, gb)]
    out, lse = net_ops.attention_with_lse(*dev[:3], causal=True)
    _, gk, gv = net_ops.attention_grad(dev[3], *dev[:3], out, lse, causal=True)
    gk, gv = gk[0, :, 0].cpu(), gv[0, :, 0].cpu()
    assert bool(gv[:21, 60].isnan().all()) and bool(gv[21:].isfinite().all())
    assert bool(gv[:21, :60].isfinite().all())
    assert bool(gk[:21].isnan().all()) and bool(gk[21:].isfinite().all())


def test_two_graphs_and_two_streams(device):
    """Two graphs captured one after the other hold workspaces of their own; replayed on two streams
    at once, with eager calls between, each has its own results."""
    g = gen(21)
    sets = [tuple(t[None].to(device) for t in inputs(g, n, 3000, 4, 2, 64, torch.bfloat16))
            for n in (1, 70)]

    def step(q, k, v, go):
        out, lse = net_ops.attention_with_lse(q, k, v, causal=True)
        return (out, lse, *net_ops.attention_grad(go, q, k, v, out, lse, causal=True))

    want = [step(*s) for s in sets]
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(*s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for h in held:
            for t in h:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        step(*sets[0])
        torch.cuda.synchronize()
        for w, h in zip(want, held):
            assert all(torch.equal(a, b) for a, b in zip(w, h))


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_that_start_anywhere(device, dtype):
    """Pointers and strides off 16 bytes, k's rows broadcast over the sequences, heads before rows:
    the same bits as from contiguous copies."""
    g = gen(33)
    lq, lk, heads, dim = 77, 140, 4, 64
    base = randn(g, 2, heads, lk + 2, dim + 3, dtype=dtype).to(device)
    q = randn(g, 2, lq, heads, dim + 1, dtype=dtype).to(device)[..., 1:]
    k = base[:1, :2, 1:lk + 1, 2:dim + 2].transpose(1, 2).expand(2, lk, 2, dim)
    v = base[:, 2:, 2:, 3:].transpose(1, 2)
    go = randn(g, 2, lq, heads, dim, dtype=dtype).to(device)  # (its strides are refused)

    def step(q, k, v, go):
        out, lse = net_ops.attention_with_lse(q, k, v, causal=True)
        return (out, lse, *net_ops.attention_grad(go, q, k, v, out, lse, causal=True))

    a = step(q, k, v, go)
    b = step(*(t.contiguous() for t in (q, k, v, go)))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradients_of_any_layout_under_autograd(device):
    """An expanded gradient and a transposed one are those of their contiguous copies; k and v shared
    by all sequences get the sum of theirs."""
    g = gen(41)
    q = randn(g, 3, 50, 4, 32, dtype=torch.float32).to(device).requires_grad_()
    k, v = (randn(g, 1, 60, 2, 32, dtype=torch.float32).to(device).requires_grad_()
            for _ in range(2))
    w = randn(g, 3, 4, 32, 50, dtype=torch.float32).to(device)

    def run(loss):
        out = net_ops.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1))
        return torch.autograd.grad(loss(out), (q, k, v))

    def by_hand(grad):
        ke, ve = (t.detach().expand(3, -1, -1, -1) for t in (k, v))
        out, lse = net_ops.attention_with_lse(q.detach(), ke, ve)
        gq, gk, gv = net_ops.attention_grad(grad.contiguous(), q.detach(), ke, ve, out, lse)
        return gq, gk.sum(0, keepdim=True), gv.sum(0, keepdim=True)

    for loss, grad in ((lambda o: o.sum(), torch.ones_like(q)),
                       (lambda o: (o.permute(0, 2, 3, 1) * w).sum(), w.permute(0, 3, 1, 2))):
        assert all(torch.equal(a, b) for a, b in zip(run(loss), by_hand(grad)))


def test_nothing_to_attend_to(device):
    """Sequences of no queries, of no keys, a batch of none, and rows of no sequence."""
    for dtype in DTYPES:
        q = torch.ones(2, 3, 2, 16, dtype=dtype, device=device, requires_grad=True)
        none = torch.empty(2, 0, 2, 16, dtype=dtype, device=device, requires_grad=True)
        out, lse = net_ops.attention_with_lse(q, none, none)
        assert not bool(out.any()) and bool((lse == -math.inf).all())
        gq, gk, gv = net_ops.attention_grad(torch.ones_like(out), q, none, none, out, lse)
        assert not bool(gq.any()) and gk.shape == none.shape
        out = net_ops.attention(none, q, q)
        assert out.shape == none.shape
        gk = torch.autograd.grad(out.sum(), q)[0]
        assert not bool(gk.any())
        starts = torch.zeros(1, dtype=torch.int32, device=device)
        rows = torch.ones(5, 2, 16, dtype=dtype, device=device)
        out, lse = net_ops.attention_with_lse(rows, rows, rows, q_starts=starts)
        assert not bool(out.any()) and bool((lse == -math.inf).all())
        assert not any(bool(t.any()) for t in net_ops.attention_grad(rows, rows, rows, rows, out, lse,
                                                                      q_starts=starts))
