"""The policy network's operators refuse what they cannot take before any launch, and give shapes
on meta tensors: through the torch operators and through the C ABI (pointers that nothing reads)."""
import ctypes
import os
import re

import pytest
import torch

from omoknuni_quantum_amd import _lib, net_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "omq_net_ops.h")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_and_binding_name_the_same_functions():
    calls = {name: args.count(",") + (args.strip() != "void")
             for name, args in re.findall(r"\b(omq_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", _text())}
    assert calls == {n: len(a) for n, (_, a) in _lib.NET_SIGNATURES.items()}
    lib = _lib.load_net()
    assert lib.omq_net_abi_version() == _lib.NET_ABI_VERSION
    assert f"#define OMQ_NET_ABI_VERSION {_lib.NET_ABI_VERSION}\n" in _text()
    assert ctypes.sizeof(_lib.OmqPolicyRows) == 12 * 8 + 6 * 4
    assert _lib.OmqPolicyRows.dtype.offset == 96


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_host_tensors_refused():
    x, w, i = torch.zeros(2, 8), torch.zeros(8), torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2)
    for call in (lambda: net_ops.token_embedding(i, x),
                 lambda: net_ops.token_embedding_grad(x, i, 4),
                 lambda: net_ops.dropout(x, 0.5, 1),
                 lambda: net_ops.add_rms_norm(x, x, w),
                 lambda: net_ops.add_rms_norm_fp8(x, x, w),
                 lambda: net_ops.add_rms_norm_grad(x, x, x, w),
                 lambda: net_ops.clipped_policy_loss(x, i, f, f),
                 lambda: net_ops.clipped_policy_loss_with_grad(x, i, f, f)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_meta_shapes():
    i = _meta(3, 5, dtype=torch.int64)
    assert net_ops.token_embedding(i, _meta(7, 4, dtype=torch.half)).shape == (3, 5, 4)
    g = net_ops.token_embedding_grad(_meta(3, 5, 4, dtype=torch.half), i, 7, 1.0, torch.float32)
    assert g.shape == (7, 4) and g.dtype == torch.float32
    x, w = _meta(3, 5, 300, dtype=torch.bfloat16), _meta(300)
    y, h = net_ops.add_rms_norm(x, x, w)
    assert y.shape == h.shape == x.shape and y.dtype == x.dtype
    q, s, h = net_ops.add_rms_norm_fp8(x, x, w, group=128)
    assert q.shape == h.shape == x.shape and s.shape == (3, 5, 3)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    assert net_ops.add_rms_norm_fp8(x, None, w)[1].shape == (3, 5, 1)
    gx, gr, gw = net_ops.add_rms_norm_grad(x, None, x, w, p=0.1)
    assert gx.shape == gr.shape == x.shape and gw.shape == w.shape and gw.dtype == w.dtype
    z, f = _meta(6, 9, dtype=torch.half), _meta(6)
    out = net_ops.clipped_policy_loss_with_grad(z, _meta(6, dtype=torch.int32), f, f)
    assert [t.shape for t in out] == [(6,), (6,), (6,), (6, 9)] and out[3].dtype == torch.half


@pytest.mark.parametrize("call,msg", [
    (lambda: net_ops.token_embedding(_meta(3), _meta(4, 8)), "int32 or int64"),
    (lambda: net_ops.token_embedding(_meta(3, dtype=torch.int32), _meta(4)), "vocabulary"),
    (lambda: net_ops.token_embedding(_meta(3, dtype=torch.int32), _meta(8, 4).t()), "adjacent"),
    (lambda: net_ops.token_embedding(_meta(3, 4, dtype=torch.int32).t(), _meta(4, 8)),
     "contiguous"),
    (lambda: net_ops.token_embedding(_meta(3, dtype=torch.int32), _meta(4, 8).double()),
     "float32, bfloat16 or float16"),
    (lambda: net_ops.token_embedding_grad(_meta(2, 8), _meta(3, dtype=torch.int32), 4), "shape"),
    (lambda: net_ops.token_embedding_grad(_meta(3, 8), _meta(3, dtype=torch.int32), 0), "< 1"),
    (lambda: net_ops.token_embedding_grad(_meta(3, 8), _meta(3, dtype=torch.int32), 4,
                                          dtype=torch.half), "dtype"),
    (lambda: net_ops.dropout(_meta(3, 8), 1.5, 0), "outside"),
    (lambda: net_ops.dropout(_meta(3, 8), float("nan"), 0), "outside"),
    (lambda: net_ops.dropout(_meta(3, 8).t(), 0.5, 0), "contiguous"),
    (lambda: net_ops.add_rms_norm(_meta(3, 8), _meta(3, 9), _meta(8)), "residual"),
    (lambda: net_ops.add_rms_norm(_meta(3, 8), _meta(3, 8).half(), _meta(8)), "residual"),
    (lambda: net_ops.add_rms_norm(_meta(3, 8), None, _meta(9)), "weight"),
    (lambda: net_ops.add_rms_norm(_meta(3, 8), None, _meta(8).half()), "weight"),
    (lambda: net_ops.add_rms_norm(_meta(8, 3).t(), None, _meta(8)), "adjacent"),
    (lambda: net_ops.add_rms_norm(_meta(3, 5, 8)[:, 1:4], None, _meta(8)), "adjacent"),
    (lambda: net_ops.add_rms_norm_fp8(_meta(3, 8), None, _meta(8), group=64), "group"),
    (lambda: net_ops.add_rms_norm_grad(_meta(3, 8), None, _meta(4, 8), _meta(8)), "grad_y"),
    (lambda: net_ops.clipped_policy_loss(_meta(3), _meta(3, dtype=torch.int32), _meta(3),
                                         _meta(3)), "rows, actions"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(4, dtype=torch.int32), _meta(3),
                                         _meta(3)), "actions must be"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(3, dtype=torch.int32), _meta(3).half(),
                                         _meta(3)), "advantages"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(3, dtype=torch.int32), _meta(3),
                                         _meta(3), target=_meta(3, 8), ref_logp=_meta(3)),
     "exclude"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(3, dtype=torch.int32), _meta(3),
                                         _meta(3), legal=_meta(3, 8)), "legal"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(3, dtype=torch.int32), _meta(3),
                                         _meta(3), target=_meta(3, 8).half()), "target"),
    (lambda: net_ops.clipped_policy_loss(_meta(3, 8), _meta(3, dtype=torch.int32), _meta(3),
                                         _meta(3), clip_low=-0.1), "negative"),
    (lambda: net_ops.clipped_policy_loss_with_grad(_meta(3, 8), _meta(3, dtype=torch.int32),
                                                   _meta(3), _meta(3), _meta(4)), "row_weight"),
])
def test_operators_refuse(call, msg):
    with pytest.raises(RuntimeError, match=msg):
        call()


def test_c_entry_points_refuse():
    lib, e = _lib.load_net(), -1
    ptr = 8  # (never read: every call below is refused first)

    def refused(rc, text, code=e):
        assert rc == code and text in lib.omq_net_last_error().decode()

    refused(lib.omq_token_embedding(ptr, 0, 4, ptr, 8, 5, 8, 9, 1.0, ptr, None), "type")
    refused(lib.omq_token_embedding(ptr, 0, -1, ptr, 8, 5, 8, 0, 1.0, ptr, None), "tokens -1")
    refused(lib.omq_token_embedding(ptr, 0, 4, ptr, 8, 5, 1 << 21, 0, 1.0, ptr, None), "too large",
            -3)
    refused(lib.omq_token_embedding(None, 0, 4, ptr, 8, 5, 8, 0, 1.0, ptr, None), "null")
    need = lib.omq_token_embedding_grad_workspace(3000, 5, 8)
    assert need > 0 and lib.omq_token_embedding_grad_workspace(-1, 5, 8) < 0
    refused(lib.omq_token_embedding_grad(ptr, 8, 0, ptr, 0, 3000, 5, 8, 1.0, ptr, 0, ptr, need - 1,
                                         None), str(need))
    refused(lib.omq_token_embedding_grad(ptr, 8, 1, ptr, 0, 3000, 5, 8, 1.0, ptr, 2, ptr, need,
                                         None), "types")
    refused(lib.omq_token_embedding_grad(ptr, 8, 0, ptr, 0, 3000, 5, 8, 1.0, ptr, 0, ptr, need,
                                         None), "16-byte")
    refused(lib.omq_dropout(ptr, 4, 8, 0, 1.01, 0, 0, ptr, None), "outside")
    refused(lib.omq_dropout(ptr, 4, 0, 0, 0.5, 0, 0, ptr, None), "dim 0")
    big = 16385
    refused(lib.omq_add_rms_norm(ptr, big, None, 0, ptr, 0, 4, big, 0, 1e-6, 0.0, 0, 0, ptr, None,
                                 None), "16384", -3)
    refused(lib.omq_add_rms_norm(ptr, 8, None, 0, ptr, 2, 4, 8, 1, 1e-6, 0.0, 0, 0, ptr, None,
                                 None), "weight")
    refused(lib.omq_add_rms_norm_fp8(ptr, 8, None, 0, ptr, 0, 4, 8, 0, 1e-6, 32, ptr, ptr, None,
                                     None), "group")
    need = lib.omq_add_rms_norm_grad_workspace(100, 8)
    refused(lib.omq_add_rms_norm_grad(ptr, 8, None, 0, ptr, 8, ptr, 0, 100, 8, 0, 1e-6, 0.0, 0, 0,
                                      None, ptr, ptr, ptr, need - 1, None), str(need))
    refused(lib.omq_add_rms_norm_grad(ptr, 8, None, 0, ptr, 8, ptr, 0, 100, 8, 0, 1e-6, 0.5, 0, 0,
                                      None, ptr, ptr, ptr, need, None), "grad_x")
    r = _lib.OmqPolicyRows()
    r.rows, r.actions, r.logits_stride = 4, 100_000, 100_000
    r.logits = r.taken = r.advantages = r.old_logp = ptr
    need = lib.omq_clipped_policy_loss_workspace(4, 100_000)
    assert need > 0
    refused(lib.omq_clipped_policy_loss(ctypes.byref(r), ptr, ptr, ptr, None, ptr, need - 1, None),
            str(need))
    refused(lib.omq_clipped_policy_loss(ctypes.byref(r), ptr, ptr, ptr, None, ptr, need, None),
            "16-byte")
    refused(lib.omq_clipped_policy_loss(ctypes.byref(r), ptr, ptr, ptr, ptr, 16, need, None),
            "stats")
    refused(lib.omq_clipped_policy_loss_grad(ctypes.byref(r), ptr, None, ptr, None), "stats")
    refused(lib.omq_clipped_policy_loss(None, ptr, ptr, ptr, None, ptr, need, None), "null")
    r.target = r.ref_logp = ptr
    refused(lib.omq_clipped_policy_loss(ctypes.byref(r), ptr, ptr, ptr, None, ptr, need, None),
            "exclude")
    r.target, r.actions = None, 0
    refused(lib.omq_clipped_policy_loss_grad(ctypes.byref(r), ptr, None, ptr, None), "actions 0")
