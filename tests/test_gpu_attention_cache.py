"""Attention over caches whose keys times the heads of queries are more than 2^31."""
import pytest
import torch

from omoknuni_quantum_amd import net_ops
from tests.test_gpu_attention import dense
from tests.test_gpu_net_ops import gen, randn, within

pytestmark = pytest.mark.gpu


def test_many_heads_over_a_large_cache(device):
    """The rows of the last sequence lie behind 2^32 elements; it alone has keys other than 0."""
    n, room, heads, kv_heads, d, used = 9, 2**20, 256, 4, 128, 103
    assert n * room * heads > 2**31 and (n - 1) * room * kv_heads * d > 2**32 - 1
    g = gen(16)
    k = torch.zeros(n, room, kv_heads, d, dtype=torch.bfloat16, device=device)
    rows = randn(g, used, kv_heads, d, dtype=torch.bfloat16)
    k[-1, :used] = rows.to(device)
    q = randn(g, n, 1, heads, d, dtype=torch.bfloat16)
    go = randn(g, n, 1, heads, d, dtype=torch.bfloat16)
    lens = torch.full((n,), used, dtype=torch.int32, device=device)
    qd, god = q.to(device), go.to(device)
    out, lse = net_ops.attention_with_lse(qd, k, k, k_lengths=lens)
    got = net_ops.attention_grad(god, qd, k, k, out, lse, k_lengths=lens)
    want, bound = dense(q[-1], rows, rows, d**-0.5, False, go[-1])
    mine = (out[-1], lse[-1], got[0][-1], got[1][-1, :used], got[2][-1, :used])
    for name, t in zip(("out", "lse", "q", "k", "v"), mine):
        within(t, want[name], bound[name])
    assert not bool(out[:-1].any())
    for t in got[1:]:
        assert all(not bool(t[s, used:].any()) for s in range(n))


def test_a_cache_shared_by_many_sequences(device):
    """131072 keys under 256 sequences of 128 heads, one and the same in memory, of which each
    sequence has its own number in use."""
    n, room, heads, d = 256, 131072, 128, 16
    g = gen(17)
    k, v = (randn(g, room, 1, d, dtype=torch.float16) for _ in range(2))
    q = randn(g, n, 1, heads, d, dtype=torch.float16)
    lens = torch.randint(0, 3000, (n,), generator=g, dtype=torch.int32)
    lens[7], lens[200] = room, 0
    kd, vd = (t.to(device)[None].expand(n, -1, -1, -1) for t in (k, v))
    out, lse = net_ops.attention_with_lse(q.to(device), kd, vd, k_lengths=lens.to(device))
    for i in (0, 7, 130, 200, n - 1):
        used = int(lens[i])
        some = q[i][:, ::50]  # (heads)
        want, bound = dense(some, k[:used], v[:used], d**-0.5, False, some)
        within(out[i][:, ::50], want["out"], bound["out"])
        within(lse[i][:, ::50], want["lse"], bound["lse"])
