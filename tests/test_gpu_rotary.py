"""The heads' norm with rotation on the GPU against its definition in 64 bits (oracle/net_ref.py).

Tolerances, u = 2^-24.  The mean square is a sum of at most 16 products a lane and five joins: off
by 22 u relative, its root by 11 u, the inverse and the products with x and the weight 5 u more.  An
angle is off by its 64-bit product and by the rounding of at most one half turn, 2 u absolute; sine
and cosine by 4 u with it.  A rotated pair of normed values with root sum of squares n is then off by
(16 + 2 * 4 + 3) u sqrt(2) n < 48 u n.  In the gradients the pair (d) is off by 12 u n(d), and
dx = (dw - n mean(dw n)) / root by 64 u ((n(d) w) + |n| mean |dw n|) / root."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_net_ops import DTYPES, gen, randn, u, within

pytestmark = pytest.mark.gpu


def pair_norm(x, pairs, interleaved):
    """For every column the root sum of squares of its pair; a column that does not turn: |x|."""
    out = x.abs().clone()
    one = torch.arange(0, 2 * pairs, 2) if interleaved else torch.arange(pairs)
    two = one + 1 if interleaved else one + pairs
    both = torch.sqrt(x[..., one]**2 + x[..., two]**2)
    out[..., one], out[..., two] = both, both
    return out


CASES = [  # tokens, heads, kv_heads, dim, sections, weights, interleaved, first position
    (1, 32, 8, 128, (64,), True, False, 100_003),
    (7, 1, 1, 2, (1,), True, False, 0),
    (225, 4, 4, 32, (8, 8), True, False, 0),
    (50, 3, 1, 64, (10, 12, 10), False, False, 5),
    (33, 2, 2, 80, (16, 16), True, False, 0),
    (20, 5, 1, 33, (4, 5), True, False, 3),
    (20, 5, 1, 33, (4, 5), True, True, 3),
    (64, 4, 2, 128, (16, 24, 24), True, True, 0),
    (9, 2, 1, 256, (128,), True, False, 900_001),
    (9, 2, 1, 255, (60, 0, 7, 3), True, True, 12),
    (300, 2, 1, 48, (), True, False, 0),
    (2000, 1, 1, 7, (3,), False, True, -40),
    (3, 1, 1, 1, (0,), True, False, 0),
]


def case(c, dtype, w_dtype):
    tokens, heads, kv_heads, dim, sections, weighted, interleaved, first = c
    sections = sections or (0,)
    g = gen(tokens + dim)
    q, k, gq, gk = (randn(g, tokens, h, dim, dtype=dtype, scale=1.5)
                    for h in (heads, kv_heads, heads, kv_heads))
    positions = first + torch.randint(0, 2000, (tokens, len(sections)), generator=g)
    freq = net_ops.rotary_frequencies(sections, device="cpu")
    wq, wk = (torch.rand(dim, generator=g).add(0.5).to(w_dtype) if weighted else None
              for _ in range(2))
    return q, k, gq, gk, positions, freq, wq, wk, sections, interleaved


def run(device, q, k, gq, gk, positions, freq, wq, wk, sections, interleaved):
    dev = [None if t is None else t.to(device) for t in (positions, freq, wq, wk)]
    args = (*dev, 1e-6, sections, interleaved)
    q, k = q.to(device), k.to(device)
    return (net_ops.head_norm_rotary(q, k, *args),
            net_ops.head_norm_rotary_grad(gq.to(device), gk.to(device), q, k, *args))


def check(got, x, g, positions, freq, w, sections, interleaved):
    out, gx, gw = got
    args = (positions, freq, w, 1e-6, sections, interleaved)
    pairs = sum(sections)
    want = net_ref.head_norm_rotary(x, *args)
    within(out, want, 48 * u * pair_norm(want, pairs, interleaved))
    want_x, want_w = net_ref.head_norm_rotary_grad(g, x, *args)
    d = net_ref.head_norm_rotary_grad(g, x, positions, freq, None, 1e-6, sections, interleaved)[0]
    size = pair_norm(d, pairs, interleaved)
    if w is None:
        return within(gx, want_x, 12 * u * size)
    w = w.double()
    root = torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
    n = x.double() / root
    bound = 64 * u * (size * w + n.abs() * (d * w * n).abs().mean(-1, keepdim=True)) / root
    within(gx, want_x, bound)
    # a sum over tokens and heads in any order, of products off by 30 u
    within(gw, want_w, (x.shape[0] * x.shape[1] + 30) * u * (size * n.abs()).sum((0, 1)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", CASES)
def test_heads(device, dtype, c):
    for w_dtype in {dtype, torch.float32}:
        q, k, gq, gk, *rest = case(c, dtype, w_dtype)
        for it in (torch.int32, torch.int64):
            rest[0] = rest[0].to(it)
            (qo, ko), (dq, dk, dqw, dkw) = run(device, q, k, gq, gk, *rest)
            pos, freq, wq, wk, sections, inter = rest
            assert qo.dtype == dtype and (dqw is None or dqw.dtype == w_dtype)
            check((qo, dq, dqw), q, gq, pos, freq, wq, sections, inter)
            check((ko, dk, dkw), k, gk, pos, freq, wk, sections, inter)


def test_slices_and_shared_positions(device):
    """q and k as slices of one product's output, and one table of positions for a batch."""
    g = gen(2)
    b, n, h, hk, d = 3, 49, 4, 2, 32
    qkv = randn(g, b, n, h + 2 * hk, d, dtype=torch.bfloat16).to(device)
    q, k, _ = qkv.split((h, hk, hk), 2)
    cell = torch.arange(n)
    pos = torch.stack((cell // 7, cell % 7), 1).int().to(device)
    freq = net_ops.rotary_frequencies((8, 8), device=device)
    w = torch.ones(d, device=device)
    args = (freq, w, w, 1e-6, (8, 8))
    got = net_ops.head_norm_rotary(q, k, pos, *args)
    want = net_ops.head_norm_rotary(q.contiguous(), k.contiguous(),
                                    pos.expand(b, n, 2).contiguous(), *args)
    assert got[0].shape == (b, n, h, d) and got[1].shape == (b, n, hk, d)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2)[0] for t in (q, k)]
    assert torch.equal(net_ops.head_norm_rotary(*heads_first, pos, *args)[0], want[0][0])


def test_autograd_graph_and_stream(device):
    q, k, gq, gk, pos, freq, wq, wk, sections, _ = case(CASES[2], torch.float32, torch.float32)
    q, k, gq, gk, pos, freq, wq, wk = (t.to(device) for t in (q, k, gq, gk, pos, freq, wq, wk))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    out = net_ops.head_norm_rotary(leaves[0], leaves[1], pos, freq, *leaves[2:], sections=sections)
    torch.autograd.backward(out, (gq, gk))

    def step():
        return (*net_ops.head_norm_rotary(q, k, pos, freq, wq, wk, sections=sections),
                *net_ops.head_norm_rotary_grad(gq, gk, q, k, pos, freq, wq, wk, 1e-6, sections))

    want = step()
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want[2:]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_no_tokens(device):
    q, k = torch.ones(0, 4, 32, device=device), torch.ones(0, 2, 32, device=device)
    w = torch.ones(32, device=device)
    args = (torch.zeros(0, 1, dtype=torch.int32, device=device),
            net_ops.rotary_frequencies((16,), device=device), w, w)
    assert net_ops.head_norm_rotary(q, k, *args)[0].shape == q.shape
    got = net_ops.head_norm_rotary_grad(q, k, q, k, *args)
    assert got[1].shape == k.shape and not bool(got[2].any()) and not bool(got[3].any())


def test_zero_and_huge_heads(device):
    """A head of zeros has 0 (eps keeps the root); NaN stays in its head."""
    q = torch.zeros(2, 2, 16, device=device)
    q[1, 1, 3] = float("nan")
    w = torch.ones(16, device=device)
    pos = torch.ones(2, 1, dtype=torch.int32, device=device)
    out = net_ops.head_norm_rotary(q, q, pos, net_ops.rotary_frequencies((8,), device=device), w, w)[0]
    assert not bool(out[0].any()) and not bool(out[1, 0].any()) and bool(torch.isnan(out[1, 1]).all())
