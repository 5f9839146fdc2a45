"""Expert router: top-k choice, router weights, counts and the balance loss.

The step in front of the routed experts (the reference is handed ``indices``
and ``scores``, ``src/mlx_iqk/nn.py:1-22``; here they can be made on the device
that uses them):

- :func:`route`           ``(indices, weights)`` of each token's top-k experts;
- :func:`balance_loss`    the loss that keeps experts evenly used, and the
  per-expert counts, of a choice already made;
- :func:`route_balanced`  both in one pass over the logits, as a training step
  takes them.

Scores are ``softmax`` over the experts or ``sigmoid`` of each logit. A logit
of ``-inf`` is no expert, and ``mask`` (bool, one per token) leaves whole rows
out: the places of a row without an expert hold index ``-1`` and weight 0,
which the experts' products turn into zero rows. Everything is differentiable
in ``logits`` (float32, float16 or bfloat16), once and in reverse mode: forward
mode and second derivatives are refused. Sums are float32 and joined in a fixed
order, so results repeat bit for bit.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from .kernels import IqkKernelError, IqkRuntimeError

MAX_EXPERTS = 1024
MAX_TOP_K = 32

_SCORING = {"softmax": 0, "sigmoid": 1}


def _rows(logits):
    """``logits`` as ``[tokens, experts]`` rows whose columns are adjacent."""
    experts = logits.shape[-1]
    rows = logits if logits.dim() == 2 else logits.reshape(-1, experts)
    step, inner = rows.stride()
    if inner != 1 or (step < experts and rows.shape[0] > 1):
        rows = rows.contiguous()
    return rows


def _check(logits, top_k, scoring, mask, offsets=None):
    """The call's logits as ``[tokens, experts]`` rows, its mask, offsets and scoring id."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise IqkRuntimeError("logits must be a tensor on the GPU")
    if logits.dtype not in K.DTYPE_IDS:
        raise IqkRuntimeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    K.refuse_tangent(logits, "logits")
    if logits.dim() < 1:
        raise IqkRuntimeError("logits must have an expert axis")
    experts = logits.shape[-1]
    if not 0 < experts <= MAX_EXPERTS:
        raise IqkKernelError(f"the router covers 1 to {MAX_EXPERTS} experts, got {experts}")
    if not 0 < top_k <= min(MAX_TOP_K, experts):
        raise IqkKernelError(f"top_k {top_k} is not in 1 to {min(MAX_TOP_K, experts)}")
    if scoring not in _SCORING:
        raise IqkRuntimeError(f"scoring must be one of {sorted(_SCORING)}, got {scoring!r}")
    dev = logits.device
    K.check_current(dev)
    rows = _rows(logits)
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != dev:
            raise IqkRuntimeError("mask must be a bool tensor beside the logits")
        if mask.shape != logits.shape[:-1]:
            raise IqkRuntimeError(
                f"mask {tuple(mask.shape)} does not match tokens {tuple(logits.shape[:-1])}")
        mask = mask.contiguous()
    if offsets is not None:
        if offsets.dtype != torch.int32 or offsets.device != dev or offsets.dim() != 1 \
                or offsets.numel() < 2:
            raise IqkRuntimeError("offsets must be int32 [segments + 1] beside the logits")
        offsets = offsets.contiguous()
    return rows, mask, offsets, _SCORING[scoring]


class _Route(torch.autograd.Function):
    """Choice and, with ``balance``, balance loss: one gradient kernel for both.
    ``given`` holds what is no input of the graph: the logits as rows, a choice
    already made (or None), mask and offsets; ``call`` the plain arguments."""

    @staticmethod
    def forward(ctx, logits, given, call, balance):
        ctx.set_materialize_grads(False)
        rows, indices, mask, offsets = given
        choose = indices is None
        if balance:
            indices, weights, loss, counts, ctx.slope = K.route_balanced(
                rows, mask, offsets, *call, indices, True)
            ctx.mark_non_differentiable(*((indices, counts) if choose else (counts,)))
        else:
            indices, weights = K.route(rows, mask, *call)
            loss = counts = ctx.slope = None
            ctx.mark_non_differentiable(indices)
        ctx.call = call
        ctx.save_for_backward(logits, indices, mask, offsets)
        return (indices if choose else None), weights, loss, counts

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper that refuses a second derivative costs more than the
        # kernel, and only create_graph needs it
        return (_refuse_twice if torch.is_grad_enabled() else _Route.gradient)(ctx, *grads)

    @staticmethod
    def gradient(ctx, _indices, grad_weights, grad_loss, _counts):
        logits, indices, mask, offsets = ctx.saved_tensors
        slope = None if grad_loss is None else ctx.slope
        if grad_weights is None and slope is None:
            return None, None, None, None
        grad = K.route_backward(_rows(logits), mask, offsets, *ctx.call, indices, grad_weights,
                                slope, grad_loss)
        return grad if logits.dim() == 2 else grad.view(logits.shape), None, None, None


_refuse_twice = once_differentiable(_Route.gradient)


def _shaped(logits, top_k, indices, weights):
    if logits.dim() == 2:
        return indices, weights
    shape = logits.shape[:-1] + (top_k,)
    return indices.view(shape), weights.view(shape)


def route(logits, top_k: int, *, scoring: str = "softmax", renormalize: bool = True,
          scale: float = 1.0, mask=None):
    """``(indices int32 [..., top_k], weights float32 [..., top_k])`` of ``logits
    [..., experts]``: the ``top_k`` largest in falling order (equal ones by
    index), and ``scale`` times their scores, divided by the scores' sum when
    ``renormalize``. Differentiable in ``logits`` through the weights."""
    rows, mask, _, scoring = _check(logits, top_k, scoring, mask)
    call = (top_k, scoring, renormalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _Route.apply(logits, (rows, None, mask, None), call, False)
    else:
        out = K.route(rows, mask, *call)
    return _shaped(logits, top_k, out[0], out[1])


def route_balanced(logits, top_k: int, *, scoring: str = "softmax", renormalize: bool = True,
                   scale: float = 1.0, mask=None, offsets=None):
    """``(indices, weights, loss, counts)``: :func:`route` and :func:`balance_loss`
    in one pass over the logits, forward and backward."""
    rows, mask, offsets, scoring = _check(logits, top_k, scoring, mask, offsets)
    call = (top_k, scoring, renormalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _Route.apply(logits, (rows, None, mask, offsets), call, True)
    else:
        out = K.route_balanced(rows, mask, offsets, *call)
    return *_shaped(logits, top_k, out[0], out[1]), out[2], out[3]


def balance_loss(logits, indices, *, scoring: str = "softmax", mask=None, offsets=None):
    """``(loss, counts)`` of a choice ``indices [..., top_k]``.

    Per segment ``g`` with ``N`` tokens (those that the mask leaves out, or that have
    no logit above ``-inf``, do not count), ``f_e = experts * counts_e / (top_k * N)``
    and ``P_e`` the mean over its tokens of the score normalised over the
    experts; the loss is the mean over the segments that hold a token of
    ``sum_e f_e P_e`` (1 when the experts are used evenly). ``offsets`` (int32
    ``[segments + 1]`` on the GPU, not falling) cuts the tokens, flattened, into
    segments, as packed sequences do; tokens before the first offset and from the last
    on are in none. None is one segment of all. ``counts`` is int32 ``[segments, experts]``; entries of
    ``indices`` outside the experts count for none. Differentiable in
    ``logits`` through the mean scores (a count has no gradient).
    """
    if not isinstance(indices, torch.Tensor) or not isinstance(logits, torch.Tensor) \
            or indices.dim() != logits.dim() or indices.shape[:-1] != logits.shape[:-1]:
        raise IqkRuntimeError("indices must be [..., top_k] beside logits [..., experts]")
    if indices.device != logits.device:
        raise IqkRuntimeError("indices must be on the logits' device")
    top_k = indices.shape[-1]
    rows, mask, offsets, scoring = _check(logits, top_k, scoring, mask, offsets)
    sel = K.expert_indices(indices)
    call = (top_k, scoring, True, 1.0)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, (rows, sel, mask, offsets), call, True)[2:]
    return K.route_balanced(rows, mask, offsets, *call, sel)[2:4]


__all__ = ["MAX_EXPERTS", "MAX_TOP_K", "balance_loss", "route", "route_balanced"]
