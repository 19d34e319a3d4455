"""Operators of a policy network over board tokens, and of its training on searches.

They run as HIP kernels for gfx950 (libomq_net_ops.so, C ABI in include/omq_net_ops.h), reached
through torch operators registered from C++ (libomq_net_torch.so, csrc/net_torch.cpp) on the
caller's current HIP stream:

    token_embedding(ids, weight, scale)                 a row of the table for each token, scaled
    add_rms_norm(x, residual, weight, eps, p, ...)      h = residual + dropout(x); y = rmsnorm(h)
    add_rms_norm_fp8(x, residual, weight, eps, group)   the same for serving, y in 8 bits
    dropout(x, p, seed, offset)                         dropout whose mask is never stored
    clipped_policy_loss(logits, actions, ...)           the policy loss over legal actions
    head_norm_rotary(q, k, positions, frequencies, ...) heads normed and rotated by position
    attention(q, k, v, ...)                             attention: batches, packed rows, caches
    token_logprobs(logits, tokens, legal, top)          log-probabilities, entropy, alternatives

Those that training uses (all but add_rms_norm_fp8) are differentiable; their gradients are also
functions of their own (``token_embedding_grad``, ``add_rms_norm_grad``,
``clipped_policy_loss_with_grad``, ``head_norm_rotary_grad``, ``attention_grad``,
``token_logprobs_with_grad``; dropout is its own gradient) for a program that runs its backward
pass by hand.  Every gradient is a function of its inputs alone, bit for bit: sums run in a fixed
order.  There are no second derivatives and no forward-mode ones, and none of the other functions:
those raise.

Elements are float32, bfloat16 or float16.  Sums and statistics are kept in float32, and a result
is rounded once (attention also rounds what its matrix products take).  Tensors of rows (the last
dimension) may be slices of wider ones as long as the rows' elements are adjacent and the rows
equally far apart; other arguments, and dropout's x, must be contiguous.
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
_ROTARY = torch.ops.omq_net.head_norm_rotary.default
_ROTARY_GRAD = torch.ops.omq_net.head_norm_rotary_grad.default
_ATTENTION = torch.ops.omq_net.attention.default
_ATTENTION_GRAD = torch.ops.omq_net.attention_grad.default
_LOGPROBS = torch.ops.omq_net.token_logprobs.default
_LOGPROBS_GRAD = torch.ops.omq_net.token_logprobs_grad.default
_LOGPROBS_WITH_GRAD = torch.ops.omq_net.token_logprobs_with_grad.default


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


# ---- norm and rotation of heads -------------------------------------------------------------
def rotary_frequencies(sections, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """float64 [sum of sections]: for an axis of n pairs base^(-j / n), j = 0 ... n - 1 (radians per
    unit of the position), the axes one after another."""
    parts = [float(base) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections]
    return torch.cat(parts).to(device)


class _HeadNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, q_weight, k_weight, eps, sections, interleaved):
        ctx.save_for_backward(q, k, positions, frequencies, q_weight, k_weight)
        ctx.args = eps, sections, interleaved
        return _ROTARY(q, k, positions, frequencies, q_weight, k_weight, *ctx.args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        gq, gk, gqw, gkw = _ROTARY_GRAD(_rows(grad_q), _rows(grad_k), *ctx.saved_tensors, *ctx.args)
        if ctx.saved_tensors[4] is None:
            gqw = gkw = None
        return gq, gk, None, None, gqw, gkw, None, None, None


def _sections(frequencies, sections):
    return tuple(int(n) for n in ((frequencies.numel(),) if sections is None else sections))


def head_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                     frequencies: torch.Tensor, q_weight: torch.Tensor | None = None,
                     k_weight: torch.Tensor | None = None, eps: float = 1e-6, sections=None,
                     interleaved: bool = False):
    """(q', k'): each head x of q [..., q_heads, dim] and k [..., k_heads, dim] normed,
    n = x / sqrt(mean(x^2) + eps) * weight, and its first 2 * pairs columns rotated by the token's
    position: a pair (a, b) of n becomes (a cos t - b sin t, b cos t + a sin t), t = position *
    frequency.  The columns behind them stay.

    q_weight, k_weight: [dim], of the heads' type or float32; both None: no norm.
    positions: int32 or int64 [..., axes], over all leading dimensions of q and k, or over the last
    of them (then they serve each of the dimensions before: [cells, 2] for a batch of boards).
    sections: the number of pairs that each axis turns, one axis' pairs after another's (None: one
    axis, all of `frequencies`); frequencies: float64 [their sum], see rotary_frequencies.
    Pair j is the columns (j, j + pairs), or (2j, 2j + 1) with interleaved.  The angle is formed in
    64 bits, so that far positions keep their phase.

    q and k may be slices of one product's output: a head's elements must be adjacent and the
    tokens equally far apart.  At most 256 columns and 4 axes.  Differentiable in q, k and the
    weights."""
    sections = _sections(frequencies, sections)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or
                                    (q_weight is not None and q_weight.requires_grad) or
                                    (k_weight is not None and k_weight.requires_grad)):
        return _HeadNormRotary.apply(q, k, positions, frequencies, q_weight, k_weight, float(eps),
                                     sections, bool(interleaved))
    return _ROTARY(q, k, positions, frequencies, q_weight, k_weight, eps, sections, interleaved)


def head_norm_rotary_grad(grad_q: torch.Tensor, grad_k: torch.Tensor, q: torch.Tensor,
                          k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
                          q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None, eps: float = 1e-6, sections=None,
                          interleaved: bool = False):
    """(grad_q, grad_k, grad_q_weight, grad_k_weight) of head_norm_rotary from its arguments and
    the gradients of its two results (contiguous).  The last two are None without weights."""
    sections = _sections(frequencies, sections)
    gq, gk, gqw, gkw = _ROTARY_GRAD(grad_q, grad_k, q, k, positions, frequencies, q_weight,
                                    k_weight, eps, sections, interleaved)
    return (gq, gk, gqw, gkw) if q_weight is not None else (gq, gk, None, None)


# ---- attention ------------------------------------------------------------------------------
class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_starts, k_starts, k_lengths):
        out, lse = _ATTENTION(q, k, v, scale, causal, q_starts, k_starts, k_lengths, True)
        ctx.save_for_backward(q, k, v, out, lse, q_starts, k_starts, k_lengths)
        ctx.args = scale, causal
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, q_starts, k_starts, k_lengths = ctx.saved_tensors
        gq, gk, gv = _ATTENTION_GRAD(_rows(grad), q, k, v, out, lse, *ctx.args, q_starts, k_starts,
                                     k_lengths)
        return gq, gk, gv, None, None, None, None, None


def _attention_args(q, scale, q_starts, k_starts):
    if scale is None:  # (a q without columns is refused with the other shapes)
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    return float(scale), q_starts if k_starts is None else k_starts


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None,
              causal: bool = False, q_starts: torch.Tensor | None = None,
              k_starts: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None):
    """softmax(scale * q k^T) v for each sequence and head, of q's shape.

    A batch: q [sequences, queries, q_heads, dim], k and v [sequences, keys, k_heads, dim].
    Packed sequences of different lengths: q [rows, q_heads, dim], k and v [rows, k_heads, dim];
    sequence s has the rows q_starts[s] to q_starts[s + 1] of q and k_starts[s] to k_starts[s + 1]
    of k and v (int32 [sequences + 1] on the device, not falling; k_starts None: q_starts).
    k_lengths (int32 [sequences] on the device) gives how many of a sequence's keys are in use,
    from the first: caches with room left, or a padded batch.

    q_heads is a multiple of k_heads; each run of q_heads / k_heads query heads shares a key head.
    causal: a sequence's last query sees all its keys, and each before it one key less.  A query
    that sees no key, and a row of no sequence, has 0.  What keys that are hidden from a query hold
    (infinities and NaN too) does not reach its result.  scale None: 1 / sqrt(dim).

    Scores and sums are float32; probabilities are rounded to the elements' type before they
    multiply v.  Head elements must be adjacent; other strides are free.  At most 128 columns.
    Differentiable in q, k and v (keys that are not in use have gradient 0)."""
    scale, k_starts = _attention_args(q, scale, q_starts, k_starts)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, scale, bool(causal), q_starts, k_starts, k_lengths)
    return _ATTENTION(q, k, v, scale, causal, q_starts, k_starts, k_lengths, False)[0]


def attention_with_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       scale: float | None = None, causal: bool = False,
                       q_starts: torch.Tensor | None = None, k_starts: torch.Tensor | None = None,
                       k_lengths: torch.Tensor | None = None):
    """(out, lse) of attention; lse float32, q's shape without dim: the logarithm of the sum of the
    exponentials of a row's scores (-inf where it sees no key).  For attention_grad."""
    scale, k_starts = _attention_args(q, scale, q_starts, k_starts)
    return _ATTENTION(q, k, v, scale, causal, q_starts, k_starts, k_lengths, True)


def attention_grad(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   out: torch.Tensor, lse: torch.Tensor, scale: float | None = None,
                   causal: bool = False, q_starts: torch.Tensor | None = None,
                   k_starts: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None):
    """(grad_q, grad_k, grad_v) of attention from its arguments, the gradient of out, and out and
    lse of attention_with_lse.  The gradients of the scores are rounded to the elements' type
    before they multiply q (for k they have twice its bits).

    Where a row's keys come in parts (each with an out and lse of its own, joined by the lse), a call
    for one part with the joined out and lse gives its share: grad_q of the parts add up."""
    scale, k_starts = _attention_args(q, scale, q_starts, k_starts)
    return _ATTENTION_GRAD(grad_out, q, k, v, out, lse, scale, causal, q_starts, k_starts,
                           k_lengths)


# ---- log-probabilities of tokens ------------------------------------------------------------
class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, legal, top):
        logp, entropy, top_logp, top_tokens, stats = _LOGPROBS(logits, tokens, legal, top, True)
        ctx.save_for_backward(logits, tokens, legal, stats)
        ctx.mark_non_differentiable(top_logp, top_tokens)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logp, grad_entropy, _top_logp, _top_tokens):
        grads = [None if g is None else _rows(g) for g in (grad_logp, grad_entropy)]
        return _LOGPROBS_GRAD(*ctx.saved_tensors, *grads), None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, legal: torch.Tensor | None = None,
                   top: int = 0):
    """(logp, entropy, top_logp, top_tokens) of a policy's rows.

    With logq the log-softmax of a row over its legal tokens: logp = logq[token], entropy =
    -sum e^logq logq, and the `top` (at most 32) most probable tokens with their logq, by falling
    logit and rising index among equals.  logp and entropy float32 [rows]; top_logp float32 and
    top_tokens int64 [rows, top], -inf and -1 where fewer tokens have a probability.

    logits [rows, vocabulary] float32/bfloat16/float16; tokens int32/int64 [rows]; legal bool like
    logits (None: all).  A token outside the vocabulary (padding) or not legal has logp 0, as
    clipped_policy_loss has it; a row without a legal token has 0 throughout and no alternatives.
    What the logits of illegal tokens hold is never used.  A NaN or an infinity above 0 among the
    legal ones makes the row's results NaN.  Differentiable in logits through logp and entropy (a
    policy-gradient term and an entropy bonus)."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogprobs.apply(logits, tokens, legal, int(top))
    return _LOGPROBS(logits, tokens, legal, top, False)[:4]


def token_logprobs_with_grad(logits: torch.Tensor, tokens: torch.Tensor,
                             logp_weight: torch.Tensor | None = None,
                             entropy_weight: torch.Tensor | None = None,
                             legal: torch.Tensor | None = None):
    """(logp, entropy, grad): those of token_logprobs and the gradient by the logits of
    sum(logp_weight * logp + entropy_weight * entropy) (float32 [rows] each, None: 0), for a
    program that goes on with ``logits.backward(grad)``.  One launch; rows of up to 16384 tokens
    are read once.  A row whose weights are 0 has no gradient, whatever its logits hold."""
    return _LOGPROBS_WITH_GRAD(logits, tokens, legal, logp_weight, entropy_weight)
