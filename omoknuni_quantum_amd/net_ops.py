"""Operators of a policy network over board tokens, and of its training on searches.

They run as HIP kernels for gfx950 (libomq_net_ops.so, C ABI in include/omq_net_ops.h), reached
through torch operators registered from C++ (libomq_net_torch.so, csrc/net_torch.cpp) on the
caller's current HIP stream:

    token_embedding(ids, weight, scale)                 a row of the table for each token, scaled
    add_rms_norm(x, residual, weight, eps, p, ...)      h = residual + dropout(x); y = rmsnorm(h)
    add_rms_norm_fp8(x, residual, weight, eps, group)   the same for serving, y in 8 bits
    dropout(x, p, seed, offset)                         dropout whose mask is never stored
    clipped_policy_loss(logits, actions, ...)           the policy loss over legal actions

The four that training uses are differentiable; their gradients are also functions of their own
(``token_embedding_grad``, ``add_rms_norm_grad``, ``clipped_policy_loss_with_grad``; dropout is its
own gradient) for a program that runs its backward pass by hand.  Every gradient is a function of
its inputs alone, bit for bit: sums run in a fixed order.  There are no second derivatives and no
forward-mode ones, and none of the other functions: those raise.

Elements are float32, bfloat16 or float16.  Sums and statistics are kept in float32, and a result
is rounded once.  Tensors of rows (the last dimension) may be slices of wider ones as long as the
rows' elements are adjacent and the rows equally far apart; other arguments, and dropout's x, must
be contiguous.
There is no CPU implementation: tensors must be on a HIP device, and a missing library raises.
"""
from __future__ import annotations

import os

import torch

from . import _lib

NET_TORCH_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libomq_net_torch.so")


def _load_net_torch() -> None:
    """Loads libomq_net_torch.so, after the library it links."""
    if hasattr(torch.ops.omq_net, "token_embedding"):
        return
    if not os.path.exists(NET_TORCH_PATH):
        raise _lib.LibraryNotBuilt(
            f"{NET_TORCH_PATH} is missing: run __graft_entry__.build() (or python -m "
            "omoknuni_quantum_amd.build) to compile it")
    _lib.load_net()
    torch.ops.load_library(NET_TORCH_PATH)


_load_net_torch()

# (the overloads themselves: the packets look theirs up at every call)
_EMBEDDING = torch.ops.omq_net.token_embedding.default
_EMBEDDING_GRAD = torch.ops.omq_net.token_embedding_grad.default
_DROPOUT = torch.ops.omq_net.dropout.default
_NORM = torch.ops.omq_net.add_rms_norm.default
_NORM_FP8 = torch.ops.omq_net.add_rms_norm_fp8.default
_NORM_GRAD = torch.ops.omq_net.add_rms_norm_grad.default
_LOSS = torch.ops.omq_net.clipped_policy_loss.default
_LOSS_GRAD = torch.ops.omq_net.clipped_policy_loss_grad.default
_LOSS_WITH_GRAD = torch.ops.omq_net.clipped_policy_loss_with_grad.default


def _word(x: int) -> int:
    """A 64-bit word as the operators' signed int of the same bits."""
    x = int(x) & 0xFFFFFFFFFFFFFFFF
    return x - (1 << 64) if x >> 63 else x


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A gradient that autograd gives, in a layout that the operators take."""
    return t.contiguous()


# ---- token embedding ------------------------------------------------------------------------
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = weight.shape[0], scale
        return _EMBEDDING(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, _EMBEDDING_GRAD(_rows(grad), ids, ctx.rows, ctx.scale, None), None


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids], of shape ids.shape + [dim].

    ids: int32 or int64; an id outside the table gives a row of zeros and takes no part in the
    gradient (padding).  weight: [vocabulary, dim].  Differentiable in weight."""
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, float(scale))
    return _EMBEDDING(ids, weight, scale)


def token_embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_embeddings: int,
                         scale: float = 1.0, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The gradient of token_embedding's weight, [num_embeddings, dim]: for every row the sum of
    `grad` over its tokens, in their order and in float32, times scale.  dtype: grad's (default)
    or float32."""
    return _EMBEDDING_GRAD(grad, ids, num_embeddings, scale, dtype)


# ---- dropout --------------------------------------------------------------------------------
class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.args = p, seed, offset
        return _DROPOUT(x, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _DROPOUT(_rows(grad), *ctx.args), None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """x with each element zeroed with probability p (in steps of 1/65536) and the others scaled
    by the inverse of the probability to be kept.

    The mask is a function of (seed, offset, the element's row and column along the last
    dimension) and is formed again in the backward pass; give each use of a step its own offset.
    Elements that are dropped are 0 whatever x holds there.  Differentiable in x.  (A HIP graph
    records seed and offset as they are: every replay drops the same elements.  So does every
    example under torch.vmap, which is a call on that example with the same arguments.)"""
    seed, offset = _word(seed), _word(offset)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, float(p), seed, offset)
    return _DROPOUT(x, p, seed, offset)


# ---- norm -----------------------------------------------------------------------------------
class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, p, seed, offset):
        y, h = _NORM(x, residual, weight, eps, p, seed, offset)
        if h.shape != x.shape:  # (not given: it is x)
            h = x.clone()
        ctx.save_for_backward(h, weight)
        ctx.args, ctx.has_residual = (eps, p, seed, offset), residual is not None
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_h):
        h, weight = ctx.saved_tensors
        grad_y = torch.zeros_like(h) if grad_y is None else _rows(grad_y)
        grad_h = None if grad_h is None else _rows(grad_h)
        gx, gr, gw = add_rms_norm_grad(grad_y, grad_h, h, weight, *ctx.args)
        return gx, gr if ctx.has_residual else None, gw, None, None, None, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                 eps: float = 1e-6, p: float = 0.0, seed: int = 0, offset: int = 0):
    """(y, h): h = residual + dropout(x, p, seed, offset), y = h / sqrt(mean(h^2) + eps) * weight
    along the last dimension.

    h is the residual of the next layer.  y is formed from the sum before it is rounded to h's
    type.  residual None: zeros (h is x itself where p is 0 and no gradient is recorded).
    weight: [dim], of x's type or float32.  At most 16384 columns.  Differentiable in x, residual
    and weight."""
    seed, offset = _word(seed), _word(offset)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _Norm.apply(x, residual, weight, float(eps), float(p), seed, offset)
    y, h = _NORM(x, residual, weight, eps, p, seed, offset)
    return y, (x if h.dim() != y.dim() or h.shape != y.shape else h)


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                     eps: float = 1e-6, group: int = 0):
    """(q, scales, h) for serving: add_rms_norm without dropout, y in 8 bits (float8_e4m3fn) as
    y = q * scale.

    scales: float32, x's shape with the last dimension 1 (group 0: one scale for a row) or
    ceil(dim / 128) (group 128: one for every 128 columns); a scale is the group's largest |y| /
    448, at least 2^-126.  Not differentiable: a backward pass through its results raises."""
    q, scales, h = _NORM_FP8(x, residual, weight, eps, group)
    return q, scales, (x if residual is None else h)


def add_rms_norm_grad(grad_y: torch.Tensor, grad_h: torch.Tensor | None, h: torch.Tensor,
                      weight: torch.Tensor, eps: float = 1e-6, p: float = 0.0, seed: int = 0,
                      offset: int = 0):
    """(grad_x, grad_residual, grad_weight) of add_rms_norm from its h, the gradient of y and
    that of h by its other uses (None: it has none).  Where p is 0, grad_x and grad_residual are
    one tensor."""
    gx, gr, gw = _NORM_GRAD(grad_y, grad_h, h, weight, eps, p, _word(seed), _word(offset))
    return (gr if gx.shape != gr.shape else gx), gr, gw


# ---- policy loss ----------------------------------------------------------------------------
class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, advantages, old_logp, low, high, coef, ref, target, legal):
        loss, logp, kl, stats = _LOSS(logits, actions, advantages, old_logp, low, high, coef, ref,
                                      target, legal, True)
        ctx.save_for_backward(logits, actions, advantages, old_logp, ref, target, legal, stats)
        ctx.args = low, high, coef
        ctx.mark_non_differentiable(logp, kl)
        return loss, logp, kl

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, _logp, _kl):
        logits, actions, advantages, old_logp, ref, target, legal, stats = ctx.saved_tensors
        grad = _LOSS_GRAD(logits, actions, advantages, old_logp, *ctx.args, ref, target, legal,
                          stats, _rows(grad_loss))
        return (grad,) + (None,) * 9


def clipped_policy_loss(logits: torch.Tensor, actions: torch.Tensor, advantages: torch.Tensor,
                        old_logp: torch.Tensor, clip_low: float = 0.2, clip_high: float = 0.2,
                        kl_coef: float = 0.0, ref_logp: torch.Tensor | None = None,
                        target: torch.Tensor | None = None, legal: torch.Tensor | None = None):
    """(loss, logp, kl), float32 [rows]: the clipped policy loss of each row and its parts.

    With logq the log-softmax of a row over its legal actions:
      logp = logq[action], ratio = exp(logp - old_logp)
      loss = -min(ratio * adv, clamp(ratio, 1 - clip_low, 1 + clip_high) * adv) + kl_coef * kl
      kl   = exp(ref_logp - logp) - (ref_logp - logp) - 1      against a reference, at the action
           = sum of target * (log target - logq) over the legal actions: against a search's
             policy (``MCTS.search``'s visit distribution) or any other distribution; with no
             advantage it is the cross-entropy training of a policy on searches
           = 0 with neither

    logits [rows, actions] float32/bfloat16/float16; legal [rows, actions] bool (None: all);
    actions int32/int64 [rows]; advantages, old_logp, ref_logp float32 [rows]; target float32
    [rows, actions], not together with ref_logp.  A row whose action is outside [0, actions) or
    not legal has logp 0 and only the target's kl; a row without a legal action has 0 throughout.
    A kl_coef of 0 leaves the kl out of loss and gradient, whatever it is (it may be infinite).
    What illegal actions' logits and targets hold is never used.  Differentiable in logits through
    loss; logp and kl carry no gradient."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _PolicyLoss.apply(logits, actions, advantages, old_logp, float(clip_low),
                                 float(clip_high), float(kl_coef), ref_logp, target, legal)
    return _LOSS(logits, actions, advantages, old_logp, clip_low, clip_high, kl_coef, ref_logp,
                 target, legal, False)[:3]


def clipped_policy_loss_with_grad(logits: torch.Tensor, actions: torch.Tensor,
                                  advantages: torch.Tensor, old_logp: torch.Tensor,
                                  row_weight: torch.Tensor | None = None, clip_low: float = 0.2,
                                  clip_high: float = 0.2, kl_coef: float = 0.0,
                                  ref_logp: torch.Tensor | None = None,
                                  target: torch.Tensor | None = None,
                                  legal: torch.Tensor | None = None):
    """(loss, logp, kl, grad): clipped_policy_loss and the gradient by the logits of
    sum(row_weight * loss) (row_weight float32 [rows], None: ones), for a program that goes on with
    ``logits.backward(grad)``.  One launch but for few very long rows; rows of up to 16384 actions
    (8192 with a target) are read once."""
    return _LOSS_WITH_GRAD(logits, actions, advantages, old_logp, clip_low, clip_high, kl_coef,
                           ref_logp, target, legal, row_weight)
