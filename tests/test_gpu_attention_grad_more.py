"""More of the attention's gradients on the GPU: parts of the keys with the whole row's out and lse,
float16 gradients of any size, and the launches by keys of many workgroups.  Bounds as in
test_gpu_attention.py."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops
from tests.test_gpu_attention import dense, inputs
from tests.test_gpu_net_ops import DTYPES, TINY, U, gen, randn, within

pytestmark = pytest.mark.gpu


# ---- parts of the keys ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,heads,kv_heads,dim", [(90, 4, 2, 64), (5, 2, 1, 128), (130, 2, 2, 32)])
@pytest.mark.parametrize("cuts", [(0, 60, 100), (0, 300, 301, 700), (0, 40, 40, 500)])
def test_parts_of_the_keys(device, dtype, lq, heads, kv_heads, dim, cuts):
    """With the out and lse of all keys each part gives its own share: the parts' dq add up to the
    whole (each rounded), their dk and dv are the whole's."""
    lk = cuts[-1]
    q, k, v, go = inputs(gen(lq + lk), lq, lk, heads, kv_heads, dim, dtype)
    want, bound = dense(q, k, v, dim**-0.5, False, go)
    q, k, v, go = (t[None].to(device) for t in (q, k, v, go))
    out, lse = net_ops.attention_with_lse(q, k, v)
    parts = [net_ops.attention_grad(go, q, k[:, i:j].contiguous(), v[:, i:j].contiguous(), out, lse)
             for i, j in zip(cuts, cuts[1:])]
    within(torch.cat([p[1][0] for p in parts]), want["k"], bound["k"])
    within(torch.cat([p[2][0] for p in parts]), want["v"], bound["v"])
    each = [p[0][0].cpu().double() for p in parts]
    off = (sum(each) - want["q"]).abs()
    limit = bound["q"] + sum(U[dtype] * t.abs() + TINY[dtype] for t in each) * 1.01
    assert bool((off <= limit).all()), float((off / limit).max())


# ---- float16 gradients of any size --------------------------------------------------------------
# A gradient of out times a power of two has gradients that are the same power of two times as
# large: all that is formed on the way is, if its exponents have room.  Elements in steps of 2^-6 are
# exact down to 2^-18 of them in float16.  The results may differ by a rounding each: U of the value,
# or half the least subnormal.
def steps(g, *shape):
    return (torch.randn(shape, generator=g) * 64).round().clamp(-255, 255).div(64).half()


def scaled_alike(got, base, factor):
    base = base.cpu().double() * factor
    off = (got.cpu().double() - base).abs()
    limit = 2.02 * U[torch.float16] * base.abs() + 1.01 * TINY[torch.float16] * (1 + factor)
    assert bool((off <= limit).all()), float((off / limit).max())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk,heads,kv_heads,dim", [(225, 225, 4, 2, 32), (90, 90, 2, 2, 64),
                                                      (100, 2100, 2, 1, 128), (70, 1000, 2, 2, 40)])
@pytest.mark.parametrize("log", [-18, -14, -10, -5, 5])
def test_float16_gradients_of_any_size(device, causal, lq, lk, heads, kv_heads, dim, log):
    g = gen(lq + lk)
    q, k, v, _ = (t[None].to(device) for t in inputs(g, lq, lk, heads, kv_heads, dim, torch.float16))
    go = steps(g, 1, lq, heads, dim).to(device)
    small = (go.double() * 2.0**log).half()
    assert torch.equal(small.double(), go.double() * 2.0**log)
    out, lse = net_ops.attention_with_lse(q, k, v, causal=causal)
    one = net_ops.attention_grad(go, q, k, v, out, lse, causal=causal)
    two = net_ops.attention_grad(small, q, k, v, out, lse, causal=causal)
    for a, b in zip(two, one):
        scaled_alike(a, b, 2.0**log)


def test_float16_rows_of_different_sizes(device):
    """Each query's gradient and each key head's goes by its own: neighbours 2^10 times as large do
    not take bits from them."""
    g, n, heads, dim = gen(77), 200, 4, 64
    q, k, v, _ = (t[None].to(device) for t in inputs(g, n, n, heads, heads, dim, torch.float16))
    go = steps(g, 1, n, heads, dim).to(device)
    out, lse = net_ops.attention_with_lse(q, k, v)
    one = net_ops.attention_grad(go, q, k, v, out, lse)
    rows = torch.randint(-14, 1, (1, n, 1, 1), generator=g).to(device)
    two = net_ops.attention_grad((go.double() * 2.0**rows).half(), q, k, v, out, lse)
    for i in range(n):
        scaled_alike(two[0][0, i], one[0][0, i], 2.0**int(rows[0, i]))
    by_head = torch.tensor([0, -14, -5, -10]).to(device)[:, None]
    two = net_ops.attention_grad((go.double() * 2.0**by_head).half(), q, k, v, out, lse)
    for h in range(heads):
        for a, b in zip(two, one):
            scaled_alike(a[0, :, h], b[0, :, h], 2.0**int(by_head[h]))


@pytest.mark.parametrize("lq,lk,causal", [(90, 90, True), (64, 2100, False)])
def test_float16_keys_that_bring_more_and_more(device, lq, lk, causal):
    """Slopes that grow by 2^20 along the keys, and rows without any."""
    g, dim = gen(lk), 64
    q, k, v, go = inputs(g, lq, lk, 2, 1, dim, torch.float16)
    v = (v.double() * 2.0**torch.linspace(-14, 6, lk)[:, None, None].round()).half()
    go[::3] = 0
    go = (go.double() * 2.0**-6).half()
    want, bound = dense(q, k, v, dim**-0.5, causal, go)
    q, k, v, go = (t[None].to(device) for t in (q, k, v, go))
    out, lse = net_ops.attention_with_lse(q, k, v, causal=causal)
    got = net_ops.attention_grad(go, q, k, v, out, lse, causal=causal)
    for name, t in zip(("q", "k", "v"), got):
        within(t[0], want[name], bound[name])
    assert not bool(got[0][0, ::3].any())


# ---- many workgroups by keys --------------------------------------------------------------------
def whole(device, dtype, causal, seqs, dim, packed):
    scale = dim**-0.5
    if packed:
        args = [torch.cat(t).to(device) for t in zip(*seqs)]
        starts = [torch.tensor([0] + [len(s[i]) for s in seqs]).cumsum(0).int().to(device)
                  for i in (0, 1)]
        kw = dict(causal=causal, q_starts=starts[0], k_starts=starts[1])
    else:
        args, kw = [torch.stack(t).to(device) for t in zip(*seqs)], dict(causal=causal)
    q, k, v, go = args
    out, lse = net_ops.attention_with_lse(q, k, v, **kw)
    got = [t.cpu() for t in (out, lse, *net_ops.attention_grad(go, q, k, v, out, lse, **kw))]
    at = [0, 0]
    for i, s in enumerate(seqs):
        want, bound = dense(*s[:3], scale, causal, s[3])
        for name, t in zip(("out", "lse", "q", "k", "v"), got):
            side = name in ("k", "v")
            mine = t[at[side]:at[side] + len(s[side])] if packed else t[i]
            within(mine, want[name], bound[name])
        at = [at[0] + len(s[0]), at[1] + len(s[1])]


@pytest.mark.parametrize("dtype,dim,heads", [(torch.bfloat16, 128, 4), (torch.float16, 128, 4),
                                             (torch.bfloat16, 100, 4), (torch.float16, 64, 8),
                                             (torch.float32, 64, 8)])
@pytest.mark.parametrize("sequences,length", [(5, 800), (5, 900), (3, 1600)])
def test_causal_workgroups_that_share_a_unit(device, dtype, dim, heads, sequences, length):
    """More workgroups than compute units and fewer than twice as many, an even and an odd number of
    tiles (of 128 keys): every key has its gradients."""
    g = gen(length + dim)
    seqs = [inputs(g, length, length, heads, heads, dim, dtype) for _ in range(sequences)]
    whole(device, dtype, True, seqs, dim, False)


@pytest.mark.parametrize("dtype,dim,heads", [(torch.bfloat16, 128, 4), (torch.float16, 64, 8)])
@pytest.mark.parametrize("lengths", [(700, 1, 300, 0, 1299, 900), (2000, 3, 1000, 640, 5)])
def test_packed_causal_workgroups_that_share_a_unit(device, dtype, dim, heads, lengths):
    g = gen(sum(lengths) + dim)
    seqs = [inputs(g, n, n + 7 * (n % 2), heads, heads, dim, dtype) for n in lengths]
    whole(device, dtype, True, seqs, dim, True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [100, 128])
def test_float32_keys_and_values_together(device, causal, dim):
    """Sums of 128 columns in one workgroup, where those fill the chip."""
    g = gen(dim)
    seqs = [inputs(g, 70, 520, 4, 4, dim, torch.float32) for _ in range(16)]
    whole(device, torch.float32, causal, seqs, dim, False)
