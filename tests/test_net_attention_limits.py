"""How large a cache the attention takes: what its arguments' checks refuse, without a launch."""
import pytest

from omoknuni_quantum_amd import _lib


def args(**kw):
    a = dict(sequences=256, q_len=1, k_len=131072, q=4096, k=4096, v=4096, q_heads=64, k_heads=8,
             dim=128, dtype=_lib.OMQ_NET_BF16, scale=0.5)
    return _lib.OmqAttentionArgs(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    {},  # (137 GB of keys and values)
    dict(sequences=64, k_len=2**20, q_heads=32, k_heads=1),
    dict(sequences=1, k_len=2**31 - 4096, q_heads=16, dim=8),
    dict(sequences=4096, k_len=8192, q_heads=128, k_heads=1),
    dict(q_starts=4096, k_starts=4096, q_len=256, k_len=256 * 131072),
])
def test_caches_that_fit_the_device(kw):
    """Queries are few, keys times the heads of queries 2^31 and more: no array has that many rows."""
    lib = _lib.load_net()
    a = args(**kw)
    assert a.sequences * a.k_len * a.q_heads >= 2**31
    assert lib.omq_attention_forward_workspace(a) >= 0
    assert lib.omq_attention_grad_workspace(a) > 0


@pytest.mark.parametrize("kw", [
    dict(k_len=2**31 - 4095), dict(q_len=2**31 - 4095, q_heads=1, k_heads=1, sequences=1),
    dict(q_len=2**20, q_heads=8), dict(sequences=2**26), dict(sequences=2**31, q_heads=1, k_heads=1),
])
def test_what_is_beyond(kw):
    lib = _lib.load_net()
    for call in (lib.omq_attention_forward_workspace, lib.omq_attention_grad_workspace):
        assert call(args(**kw)) == _lib.OMQ_E_LIMIT
        assert b"at most" in lib.omq_net_last_error()
