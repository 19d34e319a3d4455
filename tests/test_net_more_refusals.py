"""What the head norms, the attention and the log-probabilities refuse before any launch, and their
shapes and derivatives on meta tensors."""
import ctypes

import pytest
import torch

from omoknuni_quantum_amd import _lib, net_ops


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


I32, F64, BF = torch.int32, torch.float64, torch.bfloat16


def _rotary(q=None, k=None, positions=None, freq=None, **kw):
    return net_ops.head_norm_rotary(
        _meta(5, 4, 32) if q is None else q, _meta(5, 2, 32) if k is None else k,
        _meta(5, 1, dtype=I32) if positions is None else positions,
        _meta(16, dtype=F64) if freq is None else freq, **kw)


def _attn(q=None, k=None, v=None, **kw):
    q = _meta(2, 5, 4, 32) if q is None else q
    k = _meta(2, 7, 2, 32) if k is None else k
    return net_ops.attention(q, k, k if v is None else v, **kw)


def test_host_tensors_refused():
    x, i = torch.zeros(3, 2, 8), torch.zeros(3, 1, dtype=I32)
    f, b = torch.zeros(4, dtype=F64), torch.zeros(1, 3, 2, 8)
    for call in (lambda: net_ops.head_norm_rotary(x, x, i, f),
                 lambda: net_ops.head_norm_rotary_grad(x, x, x, x, i, f),
                 lambda: net_ops.attention(b, b, b),
                 lambda: net_ops.attention_with_lse(b, b, b),
                 lambda: net_ops.attention_grad(b, b, b, b, b, b[..., 0]),
                 lambda: net_ops.token_logprobs(x[0], i[:2, 0]),
                 lambda: net_ops.token_logprobs_with_grad(x[0], i[:2, 0])):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_meta_shapes():
    q, k = _rotary(_meta(3, 5, 4, 32, dtype=BF), _meta(3, 5, 2, 32, dtype=BF))
    assert q.shape == (3, 5, 4, 32) and k.shape == (3, 5, 2, 32) and q.dtype == BF
    w = _meta(32)
    got = net_ops.head_norm_rotary_grad(_meta(5, 4, 32), _meta(5, 2, 32), _meta(5, 4, 32),
                                        _meta(5, 2, 32), _meta(5, 1, dtype=I32),
                                        _meta(16, dtype=F64), w, w)
    assert [t.shape for t in got] == [(5, 4, 32), (5, 2, 32), (32,), (32,)]
    out, lse = net_ops.attention_with_lse(_meta(2, 5, 4, 32, dtype=BF), _meta(2, 7, 2, 32, dtype=BF),
                                          _meta(2, 7, 2, 32, dtype=BF))
    assert out.shape == (2, 5, 4, 32) and lse.shape == (2, 5, 4) and lse.dtype == torch.float32
    starts = _meta(4, dtype=I32)
    out, lse = net_ops.attention_with_lse(_meta(9, 4, 8), _meta(9, 4, 8), _meta(9, 4, 8),
                                          q_starts=starts)
    assert out.shape == (9, 4, 8) and lse.shape == (9, 4)
    got = net_ops.token_logprobs(_meta(6, 9, dtype=BF), _meta(6, dtype=I32), top=4)
    assert [t.shape for t in got] == [(6,), (6,), (6, 4), (6, 4)] and got[3].dtype == torch.int64
    assert net_ops.token_logprobs_with_grad(_meta(6, 9, dtype=BF), _meta(6, dtype=I32))[2].dtype == BF


@pytest.mark.parametrize("call,msg", [
    (lambda: _rotary(k=_meta(4, 2, 32)), "same tokens"),
    (lambda: _rotary(k=_meta(5, 2, 30)), "same tokens"),
    (lambda: _rotary(k=_meta(5, 2, 32, dtype=BF)), "one type"),
    (lambda: _rotary(q=_meta(5, 4, 32, dtype=F64), k=_meta(5, 2, 32, dtype=F64)), "float32, bfloat16"),
    (lambda: _rotary(q=_meta(5, 32, 4).transpose(1, 2)), "adjacent"),
    (lambda: _rotary(positions=_meta(5, 1)), "int32 or int64"),
    (lambda: _rotary(positions=_meta(4, 1, dtype=I32)), "positions"),
    (lambda: _rotary(positions=_meta(5, 2, dtype=I32)), "sections"),
    (lambda: _rotary(positions=_meta(5, 5, dtype=I32), sections=(4, 4, 4, 2, 2)), "1 to 4"),
    (lambda: _rotary(freq=_meta(16)), "float64"),
    (lambda: _rotary(freq=_meta(17, dtype=F64)), "pairs"),
    (lambda: _rotary(positions=_meta(5, 2, dtype=I32), sections=(8, 9)), "frequencies"),
    (lambda: _rotary(positions=_meta(5, 2, dtype=I32), sections=(17, -1)), "sections"),
    (lambda: _rotary(q_weight=_meta(32)), "neither"),
    (lambda: _rotary(q_weight=_meta(31), k_weight=_meta(32)), "weight"),
    (lambda: _rotary(q_weight=_meta(32, dtype=BF), k_weight=_meta(32, dtype=BF)), "weight must be"),
    (lambda: _attn(q=_meta(5, 4, 32)), "q_starts"),
    (lambda: _attn(q_starts=_meta(3, dtype=I32)), "with q_starts"),
    (lambda: _attn(k=_meta(3, 7, 2, 32)), "sequences"),
    (lambda: _attn(k=_meta(2, 7, 3, 32)), "multiple"),
    (lambda: _attn(k=_meta(2, 7, 2, 16)), "dim"),
    (lambda: _attn(v=_meta(2, 6, 2, 32)), "k and v"),
    (lambda: _attn(k=_meta(2, 7, 2, 32, dtype=BF)), "one type"),
    (lambda: _attn(k=_meta(2, 7, 32, 2).transpose(2, 3)), "adjacent"),
    (lambda: _attn(scale=0.0), "above 0"),
    (lambda: _attn(scale=-1.0), "above 0"),
    (lambda: _attn(scale=float("inf")), "above 0"),
    (lambda: _attn(scale=float("nan")), "above 0"),
    (lambda: _attn(scale=1e-60), "above 0"),
    (lambda: _attn(k_lengths=_meta(3, dtype=I32)), "k_lengths"),
    (lambda: _attn(k_lengths=_meta(2)), "k_lengths"),
    (lambda: _attn(k_starts=_meta(3, dtype=I32)), "neither"),
    (lambda: net_ops.attention(_meta(9, 2, 8), _meta(9, 2, 8), _meta(9, 2, 8),
                               q_starts=_meta(4, dtype=torch.int64)), "int32"),
    (lambda: net_ops.attention(_meta(9, 2, 8), _meta(9, 2, 8), _meta(9, 2, 8),
                               q_starts=_meta(4, dtype=I32), k_starts=_meta(5, dtype=I32)), "k_starts"),
    (lambda: net_ops.attention_grad(_meta(2, 5, 4, 16), *[_meta(2, 5, 4, 32)] * 4, _meta(2, 5, 4)),
     "grad_out"),
    (lambda: net_ops.attention_grad(*[_meta(2, 5, 4, 32)] * 5, _meta(2, 5, 3)), "lse"),
    (lambda: net_ops.attention_grad(_meta(2, 4, 5, 32).transpose(1, 2), *[_meta(2, 5, 4, 32)] * 4,
                                    _meta(2, 5, 4)), "contiguous"),
    (lambda: net_ops.token_logprobs(_meta(6), _meta(6, dtype=I32)), "vocabulary"),
    (lambda: net_ops.token_logprobs(_meta(6, 9), _meta(5, dtype=I32)), "tokens"),
    (lambda: net_ops.token_logprobs(_meta(6, 9), _meta(6)), "int32 or int64"),
    (lambda: net_ops.token_logprobs(_meta(6, 9), _meta(6, dtype=I32), _meta(6, 9)), "bool"),
    (lambda: net_ops.token_logprobs(_meta(6, 9), _meta(6, dtype=I32), top=33), "top 33"),
    (lambda: net_ops.token_logprobs(_meta(6, 9), _meta(6, dtype=I32), top=-1), "top -1"),
    (lambda: net_ops.token_logprobs_with_grad(_meta(6, 9), _meta(6, dtype=I32), _meta(5)),
     "logp_weight"),
    (lambda: net_ops.token_logprobs_with_grad(_meta(6, 9), _meta(6, dtype=I32), None,
                                              _meta(6, dtype=BF)), "entropy_weight"),
])
def test_refused(call, msg):
    with pytest.raises(RuntimeError, match=msg):
        call()


def _error(lib):
    return lib.omq_net_last_error().decode()


def test_structures_match_the_header():
    assert ctypes.sizeof(_lib.OmqRotary) == 12 * 8 + 14 * 4
    assert ctypes.sizeof(_lib.OmqAttentionArgs) == 18 * 8 + 6 * 4
    assert ctypes.sizeof(_lib.OmqLogprobRows) == 7 * 8 + 2 * 4


def test_c_refusals_of_the_rotation():
    lib, one = _lib.load_net(), 4096  # (an address that nothing reads)

    def rotary(**kw):
        r = _lib.OmqRotary(tokens=3, position_rows=3, q=one, k=one, q_token_stride=64,
                           q_head_stride=32, k_token_stride=64, k_head_stride=32, positions=one,
                           frequencies=one, q_heads=2, k_heads=2, dim=32, pairs=16, axes=1,
                           dtype=0, weight_dtype=0, eps=1e-6)
        r.section_end[0] = 16
        for name, x in kw.items():
            if name == "section_end":
                for i, e in enumerate(x):
                    r.section_end[i] = e
            else:
                setattr(r, name, x)
        return r

    E_ARG, E_LIMIT = _lib.OMQ_E_ARG, _lib.OMQ_E_LIMIT
    for kw, rc in ((dict(dtype=7), E_ARG), (dict(tokens=-1), E_ARG), (dict(q_heads=0), E_ARG),
                   (dict(pairs=17), E_ARG), (dict(axes=0), E_ARG), (dict(axes=5), E_LIMIT),
                   (dict(dim=257), E_LIMIT), (dict(tokens=2**31), E_LIMIT),
                   (dict(q_heads=40_000), E_LIMIT), (dict(section_end=[15]), E_ARG),
                   (dict(axes=2, section_end=[17, 16]), E_ARG), (dict(q_weight=one), E_ARG),
                   (dict(q_weight=one, k_weight=one, weight_dtype=1), E_ARG),
                   (dict(k_head_stride=-1), E_ARG), (dict(positions=None), E_ARG),
                   (dict(position_rows=0), E_ARG), (dict(q=None), E_ARG)):
        assert lib.omq_head_norm_rotary(rotary(**kw), one, one, None) == rc, kw
        assert "omq_head_norm_rotary" in _error(lib)
        assert lib.omq_head_norm_rotary_grad_workspace(rotary(**kw)) < 0
    assert lib.omq_head_norm_rotary(None, one, one, None) == E_ARG
    assert lib.omq_head_norm_rotary(rotary(), None, one, None) == E_ARG
    assert lib.omq_head_norm_rotary(rotary(tokens=0), None, None, None) == _lib.OMQ_OK
    w = rotary(q_weight=one, k_weight=one)
    need = lib.omq_head_norm_rotary_grad_workspace(w)
    assert need > 0 and lib.omq_head_norm_rotary_grad_workspace(rotary()) == 0
    for ws, n in ((None, need), (one, need - 1), (one + 4, need)):
        assert lib.omq_head_norm_rotary_grad(w, one, one, one, one, one, one, ws, n, None) == E_ARG
        assert "workspace" in _error(lib)
    assert lib.omq_head_norm_rotary_grad(w, one, one, one, one, None, one, one, need, None) == E_ARG


def test_c_refusals_of_the_attention():
    lib, one = _lib.load_net(), 4096

    def args(**kw):
        a = _lib.OmqAttentionArgs(sequences=2, q_len=5, k_len=7, q=one, k=one, v=one, q_heads=4,
                                  k_heads=2, dim=32, dtype=0, scale=0.5)
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    E_ARG, E_LIMIT = _lib.OMQ_E_ARG, _lib.OMQ_E_LIMIT
    for kw, rc in ((dict(dtype=3), E_ARG), (dict(q_len=-1), E_ARG), (dict(k_heads=3), E_ARG),
                   (dict(dim=0), E_ARG), (dict(dim=129), E_LIMIT), (dict(q_len=2**31), E_LIMIT),
                   (dict(sequences=2**31), E_LIMIT), (dict(q_len=2**29), E_LIMIT),
                   (dict(scale=0.0), E_ARG), (dict(scale=float("nan")), E_ARG),
                   (dict(q_starts=one), E_ARG), (dict(k_starts=one), E_ARG),
                   (dict(v_row_stride=-1), E_ARG), (dict(k=None), E_ARG), (dict(q=None), E_ARG)):
        a = args(**kw)
        assert lib.omq_attention_forward(a, one, None, None, 0, None) == rc, kw
        assert "omq_attention_forward" in _error(lib)
        assert lib.omq_attention_forward_workspace(a) < 0
        assert lib.omq_attention_grad_workspace(a) < 0
        assert lib.omq_attention_grad(a, one, one, one, one, one, one, one, 1 << 40, None) == rc
    assert lib.omq_attention_forward(None, one, None, None, 0, None) == E_ARG
    need = lib.omq_attention_forward_workspace(args())
    assert lib.omq_attention_forward(args(), None, None, one, need, None) == E_ARG
    assert lib.omq_attention_forward(args(sequences=0), None, None, None, 0, None) == _lib.OMQ_OK
    need = lib.omq_attention_grad_workspace(args())
    assert need >= 2 * 5 * 4 * 4
    for ws, n in ((None, need), (one, need - 1), (one + 8, need)):
        assert lib.omq_attention_grad(args(), one, one, one, one, one, one, ws, n, None) == E_ARG
        assert "workspace" in _error(lib)
    assert lib.omq_attention_grad(args(), one, one, one, one, None, one, one, need, None) == E_ARG


def test_c_refusals_of_the_logprobs():
    lib, one = _lib.load_net(), 4096

    def rows(**kw):
        r = _lib.OmqLogprobRows(rows=3, vocab=9, logits=one, logits_stride=9, tokens=one, dtype=0)
        for name, x in kw.items():
            setattr(r, name, x)
        return r

    E_ARG, E_LIMIT = _lib.OMQ_E_ARG, _lib.OMQ_E_LIMIT
    for kw, rc in ((dict(dtype=9), E_ARG), (dict(rows=-1), E_ARG), (dict(vocab=0), E_ARG),
                   (dict(logits_stride=-1), E_ARG), (dict(legal=one, legal_stride=-1), E_ARG),
                   (dict(rows=2**31), E_LIMIT), (dict(vocab=2**30 + 1), E_LIMIT),
                   (dict(logits=None), E_ARG), (dict(tokens=None), E_ARG)):
        assert lib.omq_token_logprobs(rows(**kw), 0, one, one, None, None, None, None) == rc, kw
        assert lib.omq_token_logprobs_grad(rows(**kw), one, None, None, one, None) == rc
        assert lib.omq_token_logprobs_with_grad(rows(**kw), None, None, one, one, one, None) == rc
        assert "omq_token_logprobs" in _error(lib)
    assert lib.omq_token_logprobs(rows(), -1, one, one, one, one, None, None) == E_ARG
    assert lib.omq_token_logprobs(rows(), 33, one, one, one, one, None, None) == E_LIMIT
    assert lib.omq_token_logprobs(rows(), 3, one, one, one, None, None, None) == E_ARG
    assert lib.omq_token_logprobs(rows(), 0, one, one, None, None, one + 4, None) == E_ARG
    assert lib.omq_token_logprobs_grad(rows(), one + 4, None, None, one, None) == E_ARG
    assert lib.omq_token_logprobs_with_grad(rows(), None, None, one, one, None, None) == E_ARG
    assert lib.omq_token_logprobs(rows(rows=0), 3, None, None, None, None, None, None) == _lib.OMQ_OK


# ---- automatic differentiation --------------------------------------------------------------
def _calls(x):
    """The functions on x [2, 3, 2, 8], each with its first result."""
    p, f = _meta(3, 1, dtype=I32), _meta(4, dtype=F64)
    o, t = _meta(2, 3, 2, 8), _meta(48, dtype=I32)
    flat = None if x is None else x.reshape(-1, 2)
    return {
        "head_norm_rotary": lambda: net_ops.head_norm_rotary(x, x, p, f)[0],
        "attention": lambda: net_ops.attention(x, x, x),
        "token_logprobs": lambda: net_ops.token_logprobs(flat, t)[0],
        "head_norm_rotary_grad": lambda: net_ops.head_norm_rotary_grad(o, o, x, x, p, f)[0],
        "attention_with_lse": lambda: net_ops.attention_with_lse(x, x, x)[0],
        "attention_grad": lambda: net_ops.attention_grad(o, x, x, x, o, _meta(2, 3, 2))[0],
        "token_logprobs_with_grad": lambda: net_ops.token_logprobs_with_grad(flat, t)[0],
    }


NAMES = list(_calls(None))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_raises(name, requires_grad):
    x = _meta(2, 3, 2, 8).requires_grad_(requires_grad)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, _meta(2, 3, 2, 8))
        with pytest.raises(NotImplementedError):
            _calls(dual)[name]()


@pytest.mark.parametrize("name", NAMES)
def test_backward_has_a_derivative_or_raises(name):
    x = _meta(2, 3, 2, 8).requires_grad_()
    out = _calls(x)[name]()
    assert out.requires_grad
    if name in NAMES[:3]:
        g, = torch.autograd.grad(out.sum(), x, create_graph=True)
        assert g.shape == x.shape
        with pytest.raises(RuntimeError):  # (no second derivative)
            g.sum().backward()
    else:
        with pytest.raises(RuntimeError, match="not implemented"):
            out.sum().backward()
    with torch.no_grad():
        assert not _calls(x)[name]().requires_grad


def test_frequencies():
    f = net_ops.rotary_frequencies((2, 3, 0), 100.0, "cpu")
    want = [1.0, 0.1, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]
    assert f.dtype == F64 and f.tolist() == pytest.approx(want, rel=1e-15)
