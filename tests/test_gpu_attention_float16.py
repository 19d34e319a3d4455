"""Attention in float16 where many keys of small probability make up a part of a row."""
import math

import pytest
import torch

from omoknuni_quantum_amd import net_ops
from tests.test_gpu_net_ops import U, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keys", [4000, 65536])
@pytest.mark.parametrize("queries", [1, 3, 200])
@pytest.mark.parametrize("above", [8.0, 12.5, 14.4])
def test_many_keys_of_small_probability(device, keys, queries, above):
    """The first key's score is `above` the others', whose share of the row is 0.05 % to 96 %: its
    value is 0 and theirs 1.  The others' probability e^-above, of the largest or of 2^8 times as
    much, has a rounding of U or of half of 2^-24 in float16 and is held times 2^7: 2^-32 of it in
    place of 2^-25.  Scores are off by 2^-24 of them (exact here but for log2 e), sums of n terms by
    (n / 32 + 32) u, for the running ones of a tile."""
    q = torch.zeros(1, queries, 1, 16, dtype=torch.float16, device=device)
    k, v = torch.zeros(2, 1, keys, 1, 16, dtype=torch.float16, device=device)
    q[..., 0], k[0, 0, 0, 0] = 1.0, above
    v[0, 1:], above = 1.0, float(k[0, 0, 0, 0])  # (rounded)
    others = (keys - 1) * math.exp(-above)
    want = others / (1 + others)
    out, lse = net_ops.attention_with_lse(q, k, v, 1.0)
    off = U[torch.float16] + 2.0**-32 * math.exp(above) + (keys / 32 + 32) * u + 4 * u * (1 + above)
    limit = want * (off + U[torch.float16]) + 2.0**-25
    assert float((out.double() - want).abs().max()) <= limit
    exact = above + math.log1p(others)
    limit = (keys / 32 + 40 + 4 * above + 4 * exact) * u
    assert float((lse.double() - exact).abs().max()) <= limit
