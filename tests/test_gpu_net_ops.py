"""The policy network's operators on the GPU against their definitions in 64 bits
(oracle/net_ref.py).

Tolerances.  U[T] is the unit roundoff of T: a result of type T is within U[T] of the float32
value it was rounded from, relative (half the least subnormal below that).  A float32 sum of n
terms added one after another is within n * u of the sum of the terms' magnitudes, u = 2^-24; the
kernels add at most a few hundred terms in a row before joining partial sums pairwise or in short
runs.  Every bound below is such a count times u times a magnitude taken from the 64-bit
reference, plus the rounding to the result's type."""
import math

import pytest
import torch

from omoknuni_quantum_amd import _lib, net_ops
from oracle import net_ref

pytestmark = pytest.mark.gpu

u = 2.0**-24
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _lib_check(rc):
    assert rc == _lib.OMQ_OK, _lib.load_net().omq_net_last_error()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def within(got, want, bound):
    """got (any type, any device) against the 64-bit `want`, |difference| <= bound + rounding."""
    dtype, got = got.dtype, got.cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    limit = bound + U[dtype] * (want.abs() + bound) + TINY[dtype]
    off = ((got - want).abs() - limit)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def strided(t, extra, device):
    """t on the device as a slice of a wider tensor whose other elements are NaN (or True)."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + extra),
                      True if t.dtype == torch.bool else float("nan"), dtype=t.dtype)
    wide[..., :t.shape[-1]] = t
    return wide.to(device)[..., :t.shape[-1]]


# ---- token embedding ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 675, 128), (225, 675, 128),
                                              (0, 5, 16), (37, 5, 3), (513, 64, 257),
                                              (1000, 1083, 1030)])
def test_embedding(device, dtype, tokens, vocab, dim):
    g = gen(tokens + dim)
    ids = torch.randint(-2, vocab + 2, (tokens,), generator=g)
    w = randn(g, vocab, dim, dtype=dtype)
    for it in (torch.int32, torch.int64):
        got = net_ops.token_embedding(ids.to(it).to(device), strided(w, 5, device), 11.3137085)
        within(got, net_ref.embedding(ids, w, 11.3137085), net_ref.embedding(ids, w, 1.0).abs() *
               11.32 * 2 * u)


def test_embedding_shapes_and_far_ids(device):
    g = gen(5)
    w = randn(g, 7, 12, dtype=torch.bfloat16)
    ids = torch.tensor([[0, 6, 2**40], [-2**40, 3, 2**31 + 1]])
    got = net_ops.token_embedding(ids.to(device), w.to(device))
    assert got.shape == (2, 3, 12)
    assert torch.equal(got.cpu().double(), net_ref.embedding(ids, w, 1.0))


GRAD_CASES = [
    # tokens, vocab, dim, skew: no tokens; one; few, listed, with rows of many tokens and of none;
    # one vocabulary row; one workgroup's sorts; radix sorts of one, two and three passes, with and
    # without a launch for the scan; tokens of few rows and rows of few tokens
    (0, 5, 16, 1), (1, 1, 1, 1), (1, 3000, 40, 1), (225, 675, 128, 1), (256, 2, 600, 1),
    (256, 20_000, 7, 2), (257, 2, 600, 1), (1024, 40, 24, 1), (1024, 1, 8, 1), (1025, 300, 129, 1),
    (1025, 200, 129, 1), (2048, 512, 600, 6), (2047, 5000, 3, 1), (2049, 5000, 48, 1),
    (2048, 400, 33, 1), (4096, 2047, 16, 1), (4096, 2048, 16, 1), (4097, 2048, 16, 1),
    (32_768, 300, 40, 1), (32_769, 300, 40, 1), (32_000, 3000, 40, 2), (4096, 1, 64, 1),
    (4096, 300, 33, 3), (4097, 3, 64, 1), (5000, 2047, 130, 1), (9000, 2048, 257, 4),
    (20_000, 70_000, 65, 3), (6000, 5_000_000, 8, 1), (50_000, 2, 513, 1), (30_001, 900, 1031, 2),
]


@pytest.mark.parametrize("tokens,vocab,dim,skew", GRAD_CASES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_grad(device, dtype, tokens, vocab, dim, skew):
    g = gen(tokens + vocab)
    ids = (torch.rand(tokens, generator=g) ** skew * vocab).long()
    ids[3::97] = -1
    ids[5::101] = vocab
    grad = randn(g, tokens, dim, dtype=dtype)
    want = net_ref.embedding_grad(grad, ids, vocab, 1.7)
    counts = net_ref.embedding_grad(torch.ones(tokens, 1), ids, vocab, 1.0)
    size = net_ref.embedding_grad(grad.abs(), ids, vocab, 1.7)
    # at most 1024 + 4096 additions in a row, and no more than there are tokens
    bound = size * u * (counts.clamp(max=6000) + 3)
    out = net_ops.token_embedding_grad(strided(grad, 3, device), ids.int().to(device), vocab, 1.7)
    assert out.dtype == dtype
    within(out, want, bound)
    wide = net_ops.token_embedding_grad(grad.to(device), ids.to(device), vocab, 1.7,
                                        torch.float32)
    within(wide, want, bound)
    # the order of the sums does not depend on the types (a scale of 2 multiplies exactly; float16
    # results of other scales come from a multiplication that rounds to float16 at once)
    two = [net_ops.token_embedding_grad(grad.to(device), ids.to(device), vocab, 2.0, t)
           for t in (None, torch.float32)]
    assert torch.equal(two[0], two[1].to(dtype))
    assert not bool(out[(counts[:, 0] == 0).to(device)].any())


def test_embedding_grad_repeats_bit_for_bit(device):
    g = gen(9)
    ids = (torch.rand(60_000, generator=g) ** 4 * 5000).int().to(device)
    grad = randn(g, 60_000, 200, dtype=torch.bfloat16).to(device)
    first = net_ops.token_embedding_grad(grad, ids, 5000, 1.0, torch.float32)
    for _ in range(3):
        assert torch.equal(first, net_ops.token_embedding_grad(grad, ids, 5000, 1.0,
                                                               torch.float32))


# ---- dropout --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(0, 8), (1, 1), (3, 8), (17, 361), (64, 130), (5, 2051)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.999999, 1.0])
def test_dropout(device, dtype, rows, dim, p):
    g = gen(rows + dim)
    x = randn(g, rows, dim, dtype=dtype)
    seed, offset = 2**64 - 3 - dim, 2**63 + 5
    got = net_ops.dropout(x.to(device), p, seed, offset)
    want = net_ref.dropout(x, p, seed, offset)
    within(got, want, want.abs() * 2 * u)
    assert torch.equal(got.cpu() != 0, (want != 0))


def test_dropped_elements_are_zero_whatever_they_hold(device):
    x = torch.full((50, 33), float("nan"))
    x[::2] = float("inf")
    keep = net_ref.keep_mask(50, 33, 0.4, 8, 1)
    got = net_ops.dropout(x.to(device), 0.4, 8, 1).cpu()
    assert torch.equal(got == 0, ~keep)
    assert bool((got[::2][keep[::2]] == float("inf")).all())
    assert bool(got[1::2][keep[1::2]].isnan().all())


def test_dropout_shape_is_rows_of_the_last_dimension(device):
    x = randn(gen(2), 3, 5, 7).to(device)
    assert torch.equal(net_ops.dropout(x, 0.3, 1).view(15, 7),
                       net_ops.dropout(x.view(15, 7), 0.3, 1))


# ---- norm -----------------------------------------------------------------------------------
NORM_SHAPES = [(0, 64), (1, 1), (3, 7), (5, 64), (33, 128), (9, 129), (7, 256), (6, 361),
               (5, 512), (4, 1000), (3, 1024), (5, 2048), (3, 2049), (2, 4096), (3, 5000),
               (2, 8192), (2, 8193), (1, 16384)]


def norm_inputs(rows, dim, dtype, w_dtype):
    g = gen(rows * 31 + dim)
    w = (torch.rand(dim, generator=g) + 0.5).to(w_dtype)
    return randn(g, rows, dim, dtype=dtype), randn(g, rows, dim, dtype=dtype, scale=2.0), w


def norm_bound(x, res, w, r):
    """h: two operations; the inverse root: a sum of at most 64 + 12 squares in a row, a root and a
    division (half the sum's relative error and two more); y: two products."""
    size = x.abs() + (0.0 if res is None else res.double().abs())
    return 3 * u * size, 60 * u * size * r * w.double().abs()


@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_norm(device, rows, dim, dtype, p):
    for w_dtype in {dtype, torch.float32}:
        x, res, w = norm_inputs(rows, dim, dtype, w_dtype)
        for residual in (res, None):
            y, h = net_ops.add_rms_norm(
                strided(x, 3, device), None if residual is None else strided(res, 9, device),
                w.to(device), 1e-5, p, 77, 5)
            want_y, want_h, r = net_ref.add_rms_norm(x, residual, w, 1e-5, p, 77, 5)
            bound_h, bound_y = norm_bound(net_ref.dropout(x, p, 77, 5), residual, w, r)
            within(h, want_h, bound_h)
            within(y, want_y, bound_y)


def test_norm_dropout_is_dropout(device):
    x, res, w = (t.to(device) for t in norm_inputs(19, 301, torch.float32, torch.float32))
    _, h = net_ops.add_rms_norm(x, res, w, 1e-6, 0.3, 4, 2)
    assert torch.equal(h, res + net_ops.dropout(x, 0.3, 4, 2))


def test_norm_rows_of_zeros_and_of_nan(device):
    x = torch.zeros(4, 200)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    x[3] = 1.0
    w = torch.ones(200)
    y, h = net_ops.add_rms_norm(x.to(device), None, w.to(device))
    assert not bool(y[0].any()) and bool(y[1].isnan().all()) and h.data_ptr() != y.data_ptr()
    assert bool(y[2, 5].isnan()) and not bool(y[3].isnan().any())
    q, s, _ = net_ops.add_rms_norm_fp8(x.to(device), None, w.to(device))
    assert float(s[0]) == 2.0**-126 and not bool(q[0].float().any())
    assert bool(q[1].float().isnan().all()) and float(s[3]) == pytest.approx(1 / 448, rel=1e-5)


@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_fp8(device, rows, dim, group, dtype):
    x, res, w = norm_inputs(rows, dim, dtype, dtype)
    q, s, h = net_ops.add_rms_norm_fp8(strided(x, 3, device), strided(res, 9, device),
                                       w.to(device), 1e-5, group)
    y, want_h, r = net_ref.add_rms_norm(x, res, w, 1e-5)
    bound_h, bound_y = norm_bound(x.double(), res, w, r)
    within(h, want_h, bound_h)
    width = group or dim
    s, q = s.cpu().double(), q.cpu().double()
    assert s.shape == (rows, -(-dim // width)) and q.shape == (rows, dim)
    for j in range(s.shape[1]):
        cols = slice(j * width, min(dim, (j + 1) * width))
        if rows == 0:
            continue
        top = y[:, cols].abs().amax(1) / 448.0
        slack = bound_y[:, cols].amax(1) / 448.0 + 3 * u * top
        assert bool(((s[:, j] - top).abs() <= slack + 2.0**-126).all())
        # e4m3: half a unit of the last of four significant bits, or of the subnormals' 2^-9
        back = q[:, cols] * s[:, j:j + 1]
        limit = y[:, cols].abs() * 2.0**-4 + s[:, j:j + 1] * 2.0**-10 + 2 * bound_y[:, cols]
        assert bool(((back - y[:, cols]).abs() <= limit).all())


@pytest.mark.parametrize("rows,dim", NORM_SHAPES + [(3000, 40), (2500, 300), (1500, 2050)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p,with_h", [(0.0, True), (0.25, False), (0.25, True)])
def test_norm_grad(device, rows, dim, dtype, p, with_h):
    if p and rows * dim > 200_000:
        p = 1.0  # (a mask that needs no Python integers: everything is dropped)
    w_dtype = torch.float32 if dim % 2 else dtype
    h, gy, w = norm_inputs(rows, dim, dtype, w_dtype)
    gh = randn(gen(dim), rows, dim, dtype=dtype) if with_h else None
    gx, gr, gw = net_ops.add_rms_norm_grad(
        strided(gy, 1, device), None if gh is None else strided(gh, 2, device),
        strided(h, 5, device), w.to(device), 1e-5, p, 3, 9)
    wx, wr, ww = net_ref.add_rms_norm_grad(gy, gh, h, w, 1e-5, p, 3, 9)
    # sums of at most 64 + 12 products in a row, and a few operations on each element
    hd, g = h.double(), gy.double() * w.double()
    r = 1.0 / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-5)
    size = r * (g.abs() + hd.abs() * r * (g * hd * r).abs().mean(-1, keepdim=True))
    if gh is not None:
        size = size + gh.double().abs()
    if rows == 0:
        size = torch.zeros(0, dim, dtype=torch.float64)
    within(gr, wr, 150 * u * size)
    scale = 1.0 if p in (0.0, 1.0) else 65536.0 / (65536 - net_ref.threshold(p))
    within(gx, wx, 150 * u * size * scale)
    assert (gx.data_ptr() == gr.data_ptr()) == (p == 0.0 or rows == 0)
    # the weight's: a row after another within a workgroup, the workgroups' sums in runs
    within(gw, ww, (rows + 120) * u * (gy.double() * hd * r).abs().sum(0))


def test_norm_grad_repeats_bit_for_bit(device):
    h, gy, w = (t.to(device) for t in norm_inputs(5000, 384, torch.bfloat16, torch.float32))
    first = net_ops.add_rms_norm_grad(gy, None, h, w)
    for _ in range(3):
        again = net_ops.add_rms_norm_grad(gy, None, h, w)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- policy loss ----------------------------------------------------------------------------
def loss_inputs(rows, actions, dtype, kl, masked, seed):
    g = gen(seed)
    z = randn(g, rows, actions, dtype=dtype, scale=3.0)
    legal = torch.rand(rows, actions, generator=g) < 0.4 if masked else None
    act = torch.randint(0, actions, (rows,), generator=g)
    if masked:
        for i in range(0, rows, 2):  # every other action is legal
            legal[i, act[i]] = True
        legal[5::7] = False
        z[~legal] = torch.finfo(dtype).min
        z[1::3][~legal[1::3]] = float("nan")
        z[2::3][~legal[2::3]] = float("inf")
    act[4::11] = -1
    act[6::13] = actions
    d = {"adv": torch.randn(rows, generator=g), "legal": legal, "z": z, "act": act,
         "weight": torch.rand(rows, generator=g)}
    ref = net_ref.policy_loss(z, act, torch.zeros(rows), torch.zeros(rows), 0.2, 0.3, 0.0,
                              legal=legal)
    d["old"] = (ref["logp"] + torch.randn(rows, generator=g) * 0.4).float()
    if kl == "sampled":
        d["ref"] = (ref["logp"] + torch.randn(rows, generator=g) * 0.4).float()
    if kl == "target":
        t = torch.randn(rows, actions, generator=g) * 2
        t[torch.rand(rows, actions, generator=g) < 0.3] = -math.inf
        t[:, 0] = 0.0
        d["target"] = torch.softmax(t, 1)
    return d


def check_loss(device, d, coef, low=0.2, high=0.3, with_grad=True):
    dev = {k: (strided(v, 3, device) if v.dim() == 2 else v.to(device))
           for k, v in d.items() if v is not None}
    inputs = dev["z"], dev["act"], dev["adv"], dev["old"]
    args = dict(clip_low=low, clip_high=high, kl_coef=coef, ref_logp=dev.get("ref"),
                target=dev.get("target"), legal=dev.get("legal"))
    want = net_ref.policy_loss(d["z"], d["act"], d["adv"], d["old"], low, high, coef, d.get("ref"),
                               d.get("target"), d.get("legal"))
    rows, cols = d["z"].shape
    z, ok = d["z"].double(), want["prob"] > 0
    # the sum of exponentials and the target's sums: at most 64 terms in a row within a row's
    # registers, 64 * 8 within a span, then short joins; exponents relative to the largest
    terms = 120 if cols <= 16384 else 800
    top = torch.where(ok, z.abs(), 0.0).amax(1) + 1.0 + math.log(cols)
    e_logp = terms * u * top
    e_ratio = want["ratio"] * (2 * e_logp + 4 * u)
    adv = d["adv"].double().abs()
    e_kl = torch.zeros(rows, dtype=torch.float64)
    if d.get("ref") is not None:
        x = torch.where(want["taken"], d["ref"].double() - want["logp"], 0.0)
        e_kl = torch.expm1(x).abs() * 2 * e_logp + 4 * u * (x.exp() + x.abs() + 1)
    if d.get("target") is not None:
        e_kl = e_logp * (1.0 + d["target"].double().sum(1)) * 2
    outs = [net_ops.clipped_policy_loss(*inputs, **args)]
    if with_grad:
        outs.append(net_ops.clipped_policy_loss_with_grad(*inputs, dev["weight"], **args))
    for out in outs:
        within(out[1], want["logp"], e_logp)
        within(out[2], want["kl"], e_kl)
        within(out[0], want["loss"], adv * e_ratio + coef * e_kl + 4 * u * want["loss"].abs())
    if with_grad:
        grad = outs[1][3].cpu()
        # rows at a bound of the clipping may fall to either side of it
        edge = torch.minimum((want["ratio"] - (1 - low)).abs(), (want["ratio"] - (1 + high)).abs())
        sure = edge > 2 * e_ratio + 1e-9
        assert float(sure.double().mean()) > 0.9 or rows < 10
        e_slope = adv * e_ratio + coef * (e_kl + 2 * e_logp * (1 if d.get("ref") is not None else 0))
        mass = (d["target"].double().sum(1) if d.get("target") is not None else 0.0) * coef
        bound = want["prob"] * (((want["slope"].abs() + mass) * 3 * e_logp + e_slope)[:, None])
        bound[torch.arange(rows), d["act"].clamp(0, cols - 1)] += e_slope
        if d.get("target") is not None:
            bound = bound + 4 * u * coef * d["target"].double()
        w = d["weight"].double()[:, None]
        bound = w * (bound + 8 * u * want["grad"].abs())
        within(grad[sure], (want["grad"] * w)[sure], bound[sure])
        if d.get("legal") is not None:
            assert not bool(grad[~d["legal"]].any())
    return dev, args, want


@pytest.mark.parametrize("rows,actions", [(1, 1), (3, 2), (20, 9), (33, 128), (31, 225), (30, 362),
                                          (17, 513), (14, 1025), (15, 2049), (16, 4672),
                                          (14, 8193), (8, 16384), (8, 16385), (15, 50_001),
                                          (5, 70_001), (3, 131_072), (130, 65_537)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kl", ["none", "sampled", "target"])
def test_policy_loss(device, rows, actions, dtype, kl):
    for masked in (False, True):
        d = loss_inputs(rows, actions, dtype, kl, masked, rows + actions)
        check_loss(device, d, {"none": 0.0, "sampled": 0.3, "target": 1.0}[kl])


def test_policy_loss_of_rows_without_anything(device):
    z = torch.tensor([[1.0, 2.0], [float("nan")] * 2, [-math.inf] * 2, [float("nan"), 1.0],
                      [0.5, -math.inf]])
    legal = torch.tensor([[False, False], [False, False], [True, True], [False, True],
                          [True, True]])
    act, f = torch.tensor([0, 1, 0, 0, 1]), torch.ones(5)
    t = torch.tensor([[0.5, 0.5]] * 5)
    out = net_ops.clipped_policy_loss_with_grad(
        z.to(device), act.to(device), f.to(device), f.to(device), None, kl_coef=1.0,
        target=t.to(device), legal=legal.to(device))
    loss, logp, kl, grad = (x.cpu() for x in out)
    for i in (0, 1, 2):
        assert loss[i] == logp[i] == kl[i] == 0 and not bool(grad[i].any())
    # one legal action, not the one taken: its probability is 1, its target 1/2
    assert logp[3] == 0 and float(kl[3]) == pytest.approx(0.5 * math.log(0.5), rel=1e-6)
    assert not bool(grad[3].any())
    # a legal action of weight zero that the target wants: kl is infinite, the gradient finite
    assert logp[4] == -math.inf and kl[4] == math.inf and loss[4] == math.inf
    assert grad[4].tolist() == [0.5, -0.5]
    # padding: the logits are NaN, the row has no action
    for cols in (300, 20_000, 80_000):
        n = torch.full((3, cols), float("nan"))
        out = net_ops.clipped_policy_loss_with_grad(
            n.to(device), torch.full((3,), -1).to(device), f[:3].to(device), f[:3].to(device))
        assert all(not bool(x.any()) for x in out)


def test_policy_loss_nan_reaches_the_result(device):
    for cols in (100, 3000, 20_000, 80_000):
        z = torch.zeros(2, cols)
        z[1, 7] = float("nan")
        f, act = torch.ones(2, device=device), torch.zeros(2, dtype=torch.int32, device=device)
        loss, logp, _, grad = net_ops.clipped_policy_loss_with_grad(z.to(device), act, f, f)
        assert bool(loss[1].isnan()) and bool(logp[1].isnan()) and bool(grad[1].isnan().all())
        assert not bool(loss[0].isnan()) and not bool(grad[0].isnan().any())


def test_policy_loss_far_logits(device):
    """Logits about a large common value: the statistics are formed about the largest one."""
    for cols in (225, 20_000, 80_000):
        d = loss_inputs(12, cols, torch.float32, "target", False, cols)
        d["z"] = (d["z"] + 1000.0).float()
        ref = net_ref.policy_loss(d["z"], d["act"], d["adv"], d["old"], 0.2, 0.3, 1.0,
                                  target=d["target"])
        out = net_ops.clipped_policy_loss(d["z"].to(device), d["act"].to(device),
                                          d["adv"].to(device), d["old"].to(device),
                                          kl_coef=1.0, target=d["target"].to(device))
        # z - max is exact to 2^-24 of 30, not of 1000
        within(out[2], ref["kl"], 800 * u * 50.0)


def test_policy_loss_many_rows_of_long_logits(device):
    """More rows than a grid dimension holds."""
    rows, cols = 70_000, 16_385
    z = torch.zeros(rows, cols, dtype=torch.bfloat16, device=device)
    act = (torch.arange(rows, device=device) % cols).int()
    f = torch.ones(rows, device=device)
    loss, logp, _ = net_ops.clipped_policy_loss(z, act, f, -math.log(cols) * f)
    assert float((logp + math.log(cols)).abs().max()) < 1e-4
    assert float((loss + 1.0).abs().max()) < 1e-3


# ---- offsets past 32 bits, streams, graphs, autograd ----------------------------------------
def test_offsets_past_32_bits(device):
    rows, dim = 2**21 + 3, 1032  # 2.16e9 elements
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=device)
    x[-1] = torch.arange(dim, device=device, dtype=torch.bfloat16)
    w = torch.ones(dim, dtype=torch.bfloat16, device=device)
    y, _ = net_ops.add_rms_norm(x, None, w)
    last = x[-1:].clone()
    assert torch.equal(y[-1:], net_ops.add_rms_norm(last, None, w)[0])
    del y
    d = net_ops.dropout(x, 0.5, 3)
    quads = dim // 4
    key = net_ref.splitmix64(net_ref.splitmix64(3) ^ 0)
    for c in (1, 500, dim - 1):
        word = net_ref.splitmix64(
            (key + net_ref.GOLDEN * ((rows - 1) * quads + c // 4)) & net_ref.M64)
        keep = (word >> (16 * (c % 4)) & 0xFFFF) >= 32768
        assert float(d[-1, c]) == (2.0 * float(x[-1, c]) if keep else 0.0)
    del d
    ids = torch.tensor([rows - 1, 0, rows - 2], device=device)
    assert torch.equal(net_ops.token_embedding(ids, x)[0], x[-1])
    tokens = torch.full((rows,), 5, dtype=torch.int32, device=device)
    tokens[-1] = 2
    grad = net_ops.token_embedding_grad(x, tokens, 7)
    assert torch.equal(grad[2], x[-1]) and not bool(grad[5].any())


def test_more_threads_than_a_grid_dimension_holds(device):
    """2^32 lanes of eight elements and more: the grid goes on along y."""
    lib = _lib.load_net()
    rows, dim = 2**29 + 5, 64
    x = torch.empty(rows * dim, dtype=torch.bfloat16, device=device)
    x[:64 * dim] = 1.0
    x[-64 * dim:] = 1.0
    _lib_check(lib.omq_dropout(x.data_ptr(), rows, dim, _lib.OMQ_NET_BF16, 0.5, 11, 3,
                               x.data_ptr(), _lib.raw_stream(x.device)))
    key = net_ref.splitmix64(net_ref.splitmix64(11) ^ 3)
    for first in (0, rows - 64):
        got = x[first * dim:(first + 64) * dim].float().cpu().view(64, dim)
        for r, c in ((0, 0), (63, 63), (40, 17)):
            word = net_ref.splitmix64(
                (key + net_ref.GOLDEN * ((first + r) * 16 + c // 4)) & net_ref.M64)
            assert float(got[r, c]) == (2.0 if word >> (16 * (c % 4)) & 0xFFFF >= 32768 else 0.0)


def test_another_stream(device):
    g = gen(3)
    x = randn(g, 4000, 512, dtype=torch.bfloat16).to(device)
    ids = torch.randint(0, 300, (4000,), generator=g).to(device)
    w = torch.ones(512, dtype=torch.bfloat16, device=device)
    want = net_ops.add_rms_norm(x, x, w), net_ops.token_embedding_grad(x, ids, 300)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = net_ops.add_rms_norm(x, x, w), net_ops.token_embedding_grad(x, ids, 300)
    s.synchronize()
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[1], want[1])


def test_graph_replays(device):
    """A training step's operators captured once; every replay against the eager result."""
    g = gen(4)
    ids = torch.randint(0, 500, (6000,), generator=g).int().to(device)
    table = randn(g, 500, 200).to(device)
    w = torch.rand(200, generator=g).to(device)
    # (spans, joined, and an element-wise gradient)
    z, act = randn(g, 64, 70_000).to(device), torch.randint(0, 70_000, (64,), generator=g).to(device)
    f = torch.ones(64, device=device)

    def step():
        e = net_ops.token_embedding(ids, table, 2.0)
        y, h = net_ops.add_rms_norm(e, e, w, 1e-6, 0.1, 5, 6)
        gx, _, gw = net_ops.add_rms_norm_grad(y, h, h, w, 1e-6, 0.1, 5, 6)
        return (y, gw, net_ops.token_embedding_grad(gx, ids, 500, 2.0),
                *net_ops.clipped_policy_loss_with_grad(z, act, f, -f))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        table.copy_(randn(g, 500, 200).to(device))
        z.copy_(randn(g, 64, 70_000).to(device))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_autograd_is_the_gradient_operators(device):
    g = gen(6)
    table = randn(g, 50, 96).to(device).requires_grad_()
    ids = torch.randint(0, 50, (4, 30), generator=g).to(device)
    res = randn(g, 4, 30, 96).to(device).requires_grad_()
    w = (torch.rand(96, generator=g) + 0.5).to(device).requires_grad_()
    up_y, up_h = randn(g, 4, 30, 96).to(device), randn(g, 4, 30, 96).to(device)
    e = net_ops.token_embedding(ids, table, 3.0)
    d = net_ops.dropout(e, 0.2, 1, 2)
    y, h = net_ops.add_rms_norm(d, res, w, 1e-6, 0.3, 1, 3)
    got = torch.autograd.grad((y, h), (table, res, w), (up_y, up_h))
    gx, gr, gw = net_ops.add_rms_norm_grad(up_y, up_h, h.detach(), w.detach(), 1e-6, 0.3, 1, 3)
    want = net_ops.token_embedding_grad(net_ops.dropout(gx, 0.2, 1, 2), ids, 50, 3.0), gr, gw
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # only one of the outputs used; no residual
    x = randn(g, 7, 96).to(device).requires_grad_()
    y, h = net_ops.add_rms_norm(x, None, w)
    only_h, = torch.autograd.grad(h.sum(), x, retain_graph=True)
    assert torch.equal(only_h, torch.ones_like(x))
    gx, = torch.autograd.grad(y, x, up_y[0, :7])
    assert torch.equal(gx, net_ops.add_rms_norm_grad(up_y[0, :7], None, x.detach(), w.detach())[0])


@pytest.mark.parametrize("cols", [225, 20_000, 80_000])
def test_policy_loss_autograd(device, cols):
    d = loss_inputs(40, cols, torch.float32, "target", True, 12)
    dev = {k: v.to(device) for k, v in d.items()}
    z = dev["z"].clone().requires_grad_()
    args = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.5, target=dev["target"], legal=dev["legal"])
    loss, logp, kl = net_ops.clipped_policy_loss(z, dev["act"], dev["adv"], dev["old"], **args)
    assert not logp.requires_grad and not kl.requires_grad
    (loss * dev["weight"]).sum().backward()
    out = net_ops.clipped_policy_loss_with_grad(dev["z"], dev["act"], dev["adv"], dev["old"],
                                                dev["weight"], **args)
    assert torch.equal(loss, out[0]) and torch.equal(z.grad, out[3])


def test_gradients_are_the_differences(device):
    """The kernels' gradients against central differences of the 64-bit definitions."""
    g = gen(8)
    d = loss_inputs(30, 60, torch.float32, "target", True, 21)
    z = torch.where(d["legal"], d["z"], 0.0)  # (finite, for the differences)
    v = randn(g, 30, 60).double()
    args = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.5, target=d["target"], legal=d["legal"])

    def value(t):
        return (net_ref.policy_loss(t, d["act"], d["adv"], d["old"], **args)["loss"] *
                d["weight"].double()).sum()

    dev = {k: (t.to(device) if isinstance(t, torch.Tensor) else t) for k, t in args.items()}
    grad = net_ops.clipped_policy_loss_with_grad(z.to(device), d["act"].to(device),
                                                 d["adv"].to(device), d["old"].to(device),
                                                 d["weight"].to(device), **dev)[3]
    step = 1e-5
    slope = float(value(z.double() + step * v) - value(z.double() - step * v)) / (2 * step)
    got = float((grad.cpu().double() * v).sum())
    assert got == pytest.approx(slope, rel=1e-4, abs=1e-4)

    x, res, w = norm_inputs(20, 70, torch.float32, torch.float32)
    gy, gh = randn(g, 20, 70), randn(g, 20, 70)
    h = res + x
    vx, vw = randn(g, 20, 70).double(), randn(g, 70).double()

    def norm_value(s):
        y, hh, _ = net_ref.add_rms_norm(h.double() + s * vx, None, w.double() + s * vw, 1e-6)
        return float((y * gy.double()).sum() + (hh * gh.double()).sum())

    gx, _, gw = net_ops.add_rms_norm_grad(gy.to(device), gh.to(device), h.to(device),
                                          w.to(device), 1e-6)
    got = float((gx.cpu().double() * vx).sum() + (gw.cpu().double() * vw).sum())
    slope = (norm_value(step) - norm_value(-step)) / (2 * step)
    assert got == pytest.approx(slope, rel=1e-4, abs=1e-3)
