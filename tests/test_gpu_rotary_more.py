"""More of the heads' norm with rotation on the GPU: gradients of more tokens than the workgroups that
keep the weights' sums take in one turn."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops
from oracle import net_ref
from tests.test_gpu_net_ops import gen, randn, u, within
from tests.test_gpu_rotary import pair_norm

pytestmark = pytest.mark.gpu


def plain(x, g, positions, freq, w):
    """(out, grad_x, grad_weight, the size of a turned gradient's pairs, x normed, root) of one axis'
    halves, in 64 bits, all tokens at once."""
    x, w = x.double(), w.double()
    angle = positions[:, :, None].double() * freq
    c, s, n = angle.cos(), angle.sin(), freq.shape[0]

    def turn(t, s):
        a, b = t[..., :n], t[..., n:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    root = torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    normed = x / root
    out = turn(normed * w, s)
    g = out if g is None else g.double()
    d = turn(g, -s)
    dn = d * w
    return (out, (dn - normed * (dn * normed).mean(-1, keepdim=True)) / root,
            (d * normed).sum((0, 1)), pair_norm(d, n, False), normed, root)


def test_all_at_once_is_the_definition():
    g = gen(4)
    x, go, w = randn(g, 5, 3, 8), randn(g, 5, 3, 8), torch.rand(8, generator=g) + 0.5
    pos, freq = torch.randint(0, 50, (5, 1), generator=g), torch.rand(4, generator=g).double()
    args = (pos, freq, w, 1e-6, (4,), False)
    out, gx, gw, *_ = plain(x, go, pos, freq, w)
    assert torch.allclose(out, net_ref.head_norm_rotary(x, *args), atol=1e-12)
    for a, b in zip((gx, gw), net_ref.head_norm_rotary_grad(go, x, *args)):
        assert torch.allclose(a, b, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(5003, 128, 160), (9001, 64, 2)])
def test_gradients_of_workgroups_that_take_turns(device, dtype, tokens, heads, kv_heads):
    """Tiles of four, three and eight tokens, more of them than 1024 workgroups, the last one in part.
    With the output as its own gradient the weights' sums have terms above 0 alone, so that no
    tile can be missing: a lane adds at most 16 terms, the 128 lane groups follow, and 32 slices of
    32 workgroups: 16 + 128 + 64 sums and 30 roundings of a term."""
    g = gen(tokens)
    pos = torch.randint(0, 3000, (tokens, 1), generator=g)
    freq = net_ops.rotary_frequencies((16,), device="cpu")
    x = [randn(g, tokens, h, 32, dtype=dtype) for h in (heads, kv_heads)]
    w = [torch.rand(32, generator=g) + 0.5 for _ in range(2)]
    dev = [t.to(device) for t in (*x, pos.int(), freq, *w)]
    out = net_ops.head_norm_rotary(*dev)
    got = net_ops.head_norm_rotary_grad(*out, *dev)
    for i in range(2):
        want, gx, gw, size, n, root = plain(x[i], out[i].cpu(), pos, freq, w[i])
        within(out[i], want, 48 * u * pair_norm(want, 16, False))
        dn = size * n.abs()
        bound = 64 * u * (size * w[i] + n.abs() * (dn * w[i]).mean(-1, keepdim=True)) / root
        within(got[i], gx, bound)
        within(got[2 + i], gw, (16 + 128 + 64 + 30) * u * dn.sum((0, 1)))
