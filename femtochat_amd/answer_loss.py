"""Losses over a chat model's answers on the MI355X: the clipped policy loss
with a KL term (answers sampled by the model itself) and the preference loss
(pairs of answers, one chosen over the other), forward and gradient.

They stand beside ``cross_entropy`` for the training that follows pretraining,
and take the model's logits as it does.  Per token y with log-probability lp::

    policy      r = exp(lp - old), d = ref - lp
                loss = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1)
    preference  h = beta ((lpw - refw) - (lpl - refl)), the sums over a pair's answers
                loss = -(1 - e) log sigmoid(h) - e log sigmoid(-h)

Layout: logits (answers, T, V), float32 or bfloat16, tokens (answers, T); tokens
equal to ``ignore_index`` (prompt, padding) have no loss, their logits are not
read and their gradient is zero.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels import _OnceOnly, _as_saved, _call, _check_tensor, _check_workspace, _dtype_code, _ptr
from .loss import _INDEX, _REDUCTIONS, valid_target_count

__all__ = [
    "policy_loss",
    "policy_loss_",
    "policy_loss_gradient_",
    "policy_loss_fused_",
    "PolicyLossFunction",
    "preference_loss",
    "preference_loss_",
    "preference_loss_gradient_",
    "PreferenceLossFunction",
]

_LOGITS = (torch.float32, torch.bfloat16)
_F32 = (torch.float32,)
_FUSED_BYTES = 1 << 18  # what fc_policy_loss_fused holds of a column, in whole 16-byte pieces


def _desc(logits, tokens, ignore_index, reduction, index_base, overwrite=False) -> _lib.AnswerDesc:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3:
        raise ValueError("logits must be an (answers, T, V) tensor")
    dev = logits.device
    if dev.type != "cuda":
        raise ValueError("the MI355X loss kernels need tensors on a HIP device (torch 'cuda'); there is no CPU path")
    B, T, V = logits.shape
    _check_tensor("logits", logits, (B, T, V), _LOGITS, dev)
    _check_tensor("tokens", tokens, (B, T), tuple(_INDEX), dev)
    return _lib.AnswerDesc(V, B, T, index_base, ignore_index, _INDEX[tokens.dtype], _dtype_code(logits.dtype),
                           _REDUCTIONS[reduction], _lib.FC_FLAG_OVERWRITE if overwrite else 0)


def _options(logits, tokens, old_logprobs, advantages, ref_logprobs, clip, kl) -> _lib.PolicyOptions:
    dev, shape = logits.device, tuple(tokens.shape)
    _check_tensor("old_logprobs", old_logprobs, shape, _F32, dev)
    per_answer = isinstance(advantages, torch.Tensor) and advantages.dim() == 1
    _check_tensor("advantages", advantages, shape[:1] if per_answer else shape, _F32, dev)
    if ref_logprobs is not None:
        _check_tensor("ref_logprobs", ref_logprobs, shape, _F32, dev)
    low, high = clip
    return _lib.PolicyOptions(float(low), float(high), float(kl), int(per_answer))


def _check_optional(dev, **tensors) -> None:
    for name, (t, shape) in tensors.items():
        if t is not None:
            _check_tensor(name, t, shape, _F32, dev)


def _dy(dy, dev, n: int) -> Optional[torch.Tensor]:
    """dy as n floats on the device, or None for 1."""
    if dy is None or (isinstance(dy, (int, float)) and dy == 1):
        return None
    if not isinstance(dy, torch.Tensor):
        dy = torch.full((n,), float(dy), dtype=torch.float32, device=dev)
    dy = dy.to(device=dev, dtype=torch.float32).contiguous()
    if dy.numel() != n:
        raise ValueError(f"dy must hold {n} value(s), got {dy.numel()}")
    return dy


def _held_at_once(logits: torch.Tensor) -> bool:
    """Whether fc_policy_loss_fused takes these columns: one that may begin inside a
    16-byte piece has up to a piece less one value fewer."""
    size = logits.element_size()
    n = logits.shape[-1] * size
    return n <= _FUSED_BYTES - (16 - size) or (n == _FUSED_BYTES and logits.data_ptr() % 16 == 0)


def _gradient_like(logits: torch.Tensor) -> torch.Tensor:
    """A buffer for the logits' gradient that lies like them against 16 bytes."""
    off = (logits.data_ptr() & 15) // logits.element_size()
    if off == 0:
        return torch.empty_like(logits)
    return torch.empty(logits.numel() + off, dtype=logits.dtype, device=logits.device)[off:].view(logits.shape)


# ---- the policy loss ------------------------------------------------------------


def policy_loss_(losses: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor,
                 advantages: torch.Tensor, *, ref_logprobs: Optional[torch.Tensor] = None,
                 clip: Tuple[float, float] = (0.2, 0.2), kl: float = 0.0, ignore_index: int = -1,
                 reduction: str = "mean", index_base: int = 0, logprobs: Optional[torch.Tensor] = None,
                 stats: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                 reduced: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None) -> None:
    """Per-token losses into ``losses`` (tokens' shape, float32).  ``advantages``
    are per token (answers, T) or per answer (answers,).  On request: the tokens'
    ``logprobs``, the sum or mean over the answers' tokens (``reduced``, 1 float),
    their number (``count``), and what the gradient needs: ``stats``
    (answers, T, 2) and ``weights`` (d loss / d logprob)."""
    d = _desc(logits, tokens, ignore_index, reduction, index_base)
    o = _options(logits, tokens, old_logprobs, advantages, ref_logprobs, clip, kl)
    dev, shape = logits.device, tuple(tokens.shape)
    _check_tensor("losses", losses, shape, _F32, dev)
    _check_optional(dev, logprobs=(logprobs, shape), stats=(stats, shape + (2,)), weights=(weights, shape),
                    reduced=(reduced, (1,)), count=(count, (1,)))
    _call(dev, _lib.lib().fc_policy_loss_fwd, ctypes.byref(d), ctypes.byref(o), _ptr(logits), _ptr(tokens),
          _ptr(old_logprobs), _ptr(advantages), _ptr(ref_logprobs), _ptr(losses), _ptr(logprobs), _ptr(stats),
          _ptr(weights), _ptr(reduced), _ptr(count))


def policy_loss(logits, tokens, old_logprobs, advantages, *, reduction: str = "mean", **options) -> torch.Tensor:
    """The losses (reduction "none") or their sum / mean over the answers' tokens
    (a 0-d tensor); the options of ``policy_loss_``."""
    losses = torch.empty(tokens.shape, dtype=torch.float32, device=logits.device)
    if reduction == "none":
        policy_loss_(losses, logits, tokens, old_logprobs, advantages, reduction=reduction, **options)
        return losses
    reduced = torch.empty(1, dtype=torch.float32, device=logits.device)
    policy_loss_(losses, logits, tokens, old_logprobs, advantages, reduction=reduction, reduced=reduced, **options)
    return reduced[0]


def policy_loss_gradient_(delta: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, dy, stats: torch.Tensor,
                          weights: torch.Tensor, *, ignore_index: int = -1, reduction: str = "mean",
                          index_base: int = 0, count: Optional[torch.Tensor] = None, accumulate: bool = True) -> None:
    """delta += scale w (onehot - softmax(logits)) from the forward's ``stats``
    and ``weights`` (``accumulate=False`` writes, with zeros outside the answers).
    ``dy``: a number or a device tensor (1 value; tokens' shape for "none");
    ``count`` is counted when not given for "mean"."""
    d = _desc(logits, tokens, ignore_index, reduction, index_base, overwrite=not accumulate)
    dev, shape = logits.device, tuple(tokens.shape)
    _check_tensor("delta", delta, tuple(logits.shape), (logits.dtype,), dev)
    _check_optional(dev, stats=(stats, shape + (2,)), weights=(weights, shape), count=(count, (1,)))
    dy = _dy(dy, dev, tokens.numel() if reduction == "none" else 1)
    if reduction == "mean" and count is None:
        count = _count(tokens, ignore_index)
    _call(dev, _lib.lib().fc_policy_loss_bwd, ctypes.byref(d), _ptr(delta), _ptr(logits), _ptr(tokens), _ptr(stats),
          _ptr(weights), _ptr(dy), _ptr(count))


def _count(tokens, ignore_index) -> torch.Tensor:
    with torch.cuda.device(tokens.device):
        return valid_target_count(tokens, ignore_index)


def policy_loss_fused_(losses: torch.Tensor, delta: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor,
                       old_logprobs: torch.Tensor, advantages: torch.Tensor, dy=None, *,
                       ref_logprobs: Optional[torch.Tensor] = None, clip: Tuple[float, float] = (0.2, 0.2),
                       kl: float = 0.0, ignore_index: int = -1, reduction: str = "mean", index_base: int = 0,
                       logprobs: Optional[torch.Tensor] = None, stats: Optional[torch.Tensor] = None,
                       weights: Optional[torch.Tensor] = None, reduced: Optional[torch.Tensor] = None,
                       count: Optional[torch.Tensor] = None) -> None:
    """``policy_loss_`` and its gradient (written to ``delta``, zeros outside the
    answers) with the logits read once: the loss as the step's last node.
    ``dy``: None (1), a number or a device tensor.  Columns of up to 256 KB (less
    14 bytes in bfloat16, 12 in float32, where a column may begin inside a 16-byte
    piece of memory); the library raises FC_ERR_UNSUPPORTED above."""
    d = _desc(logits, tokens, ignore_index, reduction, index_base, overwrite=True)
    o = _options(logits, tokens, old_logprobs, advantages, ref_logprobs, clip, kl)
    dev, shape = logits.device, tuple(tokens.shape)
    _check_tensor("losses", losses, shape, _F32, dev)
    _check_tensor("delta", delta, tuple(logits.shape), (logits.dtype,), dev)
    _check_optional(dev, logprobs=(logprobs, shape), stats=(stats, shape + (2,)), weights=(weights, shape),
                    reduced=(reduced, (1,)), count=(count, (1,)))
    dy = _dy(dy, dev, tokens.numel() if reduction == "none" else 1)
    if reduction == "mean" and count is None:
        count = torch.empty(1, dtype=torch.float32, device=dev)
    _call(dev, _lib.lib().fc_policy_loss_fused, ctypes.byref(d), ctypes.byref(o), _ptr(logits), _ptr(tokens),
          _ptr(old_logprobs), _ptr(advantages), _ptr(ref_logprobs), _ptr(losses), _ptr(logprobs), _ptr(stats),
          _ptr(weights), _ptr(reduced), _ptr(count), _ptr(delta), _ptr(dy))


def _save(ctx, desc, logits, tokens, room) -> None:
    ctx.save_for_backward(logits, tokens, room)
    ctx.desc, ctx.n, ctx.device = desc, tokens.numel(), logits.device
    ctx.saved_as = ((logits.shape, logits.dtype), (tokens.shape, tokens.dtype), (room.shape, room.dtype))


_SAVED = ("logits", "tokens", "statistics")


class PolicyLossFunction(torch.autograd.Function):
    """``PolicyLossFunction.apply(logits, tokens, old_logprobs, advantages,
    ref_logprobs, clip, kl, ignore_index, reduction)``: gradients for the logits
    only.  With a reduction, the forward forms the gradient of the value itself
    beside it, in one pass over the logits; the backward touches nothing where the
    incoming gradient is 1, and forms it again (rounded once, as any further backward
    through the same node does) where it is not."""

    @classmethod
    def apply(cls, logits, *args):
        # (a copy that autograd knows, so that what the node saves leads to the caller's logits)
        if isinstance(logits, torch.Tensor) and not logits.is_contiguous():
            logits = logits.contiguous()
        return super().apply(logits, *args)

    @staticmethod
    def forward(ctx, logits, tokens, old_logprobs, advantages, ref_logprobs=None, clip=(0.2, 0.2), kl=0.0,
                ignore_index=-1, reduction="mean"):
        if any(ctx.needs_input_grad[2:5]):
            raise ValueError("old_logprobs, advantages and ref_logprobs have no gradient; pass them detached")
        d = _desc(logits, tokens, ignore_index, reduction, 0, overwrite=True)
        o = _options(logits, tokens, old_logprobs, advantages, ref_logprobs, clip, kl)
        dev, n = logits.device, tokens.numel()
        # One allocation for what the backward needs and for the losses (a small step
        # is host time): stats (2 n), weights (n), losses (n), the count.
        room = torch.empty(4 * n + 1, dtype=torch.float32, device=dev)
        out = torch.empty(tokens.shape if reduction == "none" else (), dtype=torch.float32, device=dev)
        at = room.data_ptr()
        stats, weights, losses = at, at + 8 * n, at + 12 * n
        count = at + 16 * n if reduction == "mean" else None
        reduced = out.data_ptr()
        if reduction == "none":
            losses, reduced = reduced, None
        inputs = (logits.data_ptr(), tokens.data_ptr(), old_logprobs.data_ptr(), advantages.data_ptr(), _ptr(ref_logprobs),
                  losses, None, stats, weights)
        ctx.delta = None
        if ctx.needs_input_grad[0] and reduction != "none" and _held_at_once(logits):
            ctx.delta = _gradient_like(logits)
            _call(dev, _lib.lib().fc_policy_loss_fused, ctypes.byref(d), ctypes.byref(o), *inputs, reduced, count,
                  ctx.delta.data_ptr(), None)
        else:
            _call(dev, _lib.lib().fc_policy_loss_fwd, ctypes.byref(d), ctypes.byref(o), *inputs, reduced, count)
        _save(ctx, d, logits, tokens, room)
        return out

    @staticmethod
    def backward(ctx, dout):
        delta, ctx.delta = ctx.delta, None
        logits, tokens, room = _as_saved(ctx.saved_tensors, _SAVED, ctx.saved_as, ctx.device)
        dout = _as_floats(dout)
        # (copies that hooks hand back may lie otherwise against 16 bytes)
        formed = delta is not None and (delta.data_ptr() ^ logits.data_ptr()) & 15 == 0
        if not formed:
            delta = _gradient_like(logits)
        ctx.desc.flags = _lib.FC_FLAG_OVERWRITE | (_lib.FC_FLAG_FORMED if formed else 0)
        at, n = room.data_ptr(), ctx.n
        count = at + 16 * n if ctx.desc.reduction == _REDUCTIONS["mean"] else None
        _call(delta.device, _lib.lib().fc_policy_loss_bwd, ctypes.byref(ctx.desc), delta.data_ptr(), logits.data_ptr(),
              tokens.data_ptr(), at, at + 8 * n, dout.data_ptr(), count)
        if torch.is_grad_enabled():
            delta = _OnceOnly.apply("the policy loss", delta, logits, dout)
        return (delta,) + (None,) * 8


def _as_floats(dy: torch.Tensor) -> torch.Tensor:
    if dy.dtype != torch.float32:
        dy = dy.float()
    return dy if dy.is_contiguous() else dy.contiguous()


def _scale(x: torch.Tensor, dy: torch.Tensor) -> None:
    """x *= dy (one value, on the device), in place; not touched where dy is 1."""
    _call(x.device, _lib.lib().fc_scale_gradient, _ptr(x), _dtype_code(x.dtype), x.numel(), _ptr(_as_floats(dy)))


# ---- the preference loss --------------------------------------------------------


def preference_loss_(losses: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, ref_logprobs: torch.Tensor, *,
                     beta: float = 0.1, label_smoothing: float = 0.0, ignore_index: int = -1, reduction: str = "mean",
                     index_base: int = 0, rewards: Optional[torch.Tensor] = None,
                     logprobs: Optional[torch.Tensor] = None, stats: Optional[torch.Tensor] = None,
                     weights: Optional[torch.Tensor] = None, reduced: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None) -> None:
    """Per-pair losses into ``losses`` (pairs,).  The first half of the answers was
    chosen over the second half, in order; ``ref_logprobs`` (answers,) are the
    reference model's sums over each answer.  On request: ``rewards`` (answers,),
    beta times the log ratios; the tokens' ``logprobs``; the sum or mean over the
    pairs (``reduced``, 1 float); and for the gradient ``stats`` (answers, T, 2)
    and ``weights`` (answers,).  ``workspace``: answers * T float64 values,
    allocated here when not given."""
    d = _desc(logits, tokens, ignore_index, reduction, index_base)
    dev, shape = logits.device, tuple(tokens.shape)
    B = shape[0]
    if B % 2 != 0:
        raise ValueError(f"answers come in pairs, got {B}")
    _check_tensor("losses", losses, (B // 2,), _F32, dev)
    _check_tensor("ref_logprobs", ref_logprobs, (B,), _F32, dev)
    _check_optional(dev, rewards=(rewards, (B,)), logprobs=(logprobs, shape), stats=(stats, shape + (2,)),
                    weights=(weights, (B,)), reduced=(reduced, (1,)))
    o = _lib.PreferenceOptions(float(beta), float(label_smoothing))
    if workspace is None:
        workspace = torch.empty(shape, dtype=torch.float64, device=dev)
    else:
        _check_workspace(workspace, 0, dev)  # (its size is the library's to refuse)
    _call(dev, _lib.lib().fc_preference_loss_fwd, ctypes.byref(d), ctypes.byref(o), _ptr(logits), _ptr(tokens),
          _ptr(ref_logprobs), _ptr(losses), _ptr(rewards), _ptr(logprobs), _ptr(stats), _ptr(weights), _ptr(reduced),
          _ptr(workspace), workspace.numel() * workspace.element_size())


def preference_loss(logits, tokens, ref_logprobs, *, reduction: str = "mean", **options) -> torch.Tensor:
    """The losses (reduction "none", one per pair) or their sum / mean (a 0-d
    tensor); the options of ``preference_loss_``."""
    losses = torch.empty(tokens.shape[0] // 2, dtype=torch.float32, device=logits.device)
    if reduction == "none":
        preference_loss_(losses, logits, tokens, ref_logprobs, reduction=reduction, **options)
        return losses
    reduced = torch.empty(1, dtype=torch.float32, device=logits.device)
    preference_loss_(losses, logits, tokens, ref_logprobs, reduction=reduction, reduced=reduced, **options)
    return reduced[0]


def preference_loss_gradient_(delta: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, dy,
                              stats: torch.Tensor, weights: torch.Tensor, *, ignore_index: int = -1,
                              reduction: str = "mean", index_base: int = 0, accumulate: bool = True) -> None:
    """delta += scale w (onehot - softmax(logits)) from the forward's ``stats`` and
    ``weights`` (``accumulate=False`` writes, with zeros outside the answers).
    ``dy``: a number or a device tensor (1 value; one per pair for "none")."""
    d = _desc(logits, tokens, ignore_index, reduction, index_base, overwrite=not accumulate)
    dev, shape = logits.device, tuple(tokens.shape)
    if shape[0] % 2 != 0:
        raise ValueError(f"answers come in pairs, got {shape[0]}")
    _check_tensor("delta", delta, tuple(logits.shape), (logits.dtype,), dev)
    _check_tensor("stats", stats, shape + (2,), _F32, dev)
    _check_tensor("weights", weights, shape[:1], _F32, dev)
    dy = _dy(dy, dev, shape[0] // 2 if reduction == "none" else 1)
    _call(dev, _lib.lib().fc_preference_loss_bwd, ctypes.byref(d), _ptr(delta), _ptr(logits), _ptr(tokens),
          _ptr(stats), _ptr(weights), _ptr(dy))


class PreferenceLossFunction(torch.autograd.Function):
    """``PreferenceLossFunction.apply(logits, tokens, ref_logprobs, beta,
    label_smoothing, ignore_index, reduction)`` -> (loss, rewards): gradients for
    the logits, through the loss only."""

    @classmethod
    def apply(cls, logits, *args):
        # (a copy that autograd knows, so that what the node saves leads to the caller's logits)
        if isinstance(logits, torch.Tensor) and not logits.is_contiguous():
            logits = logits.contiguous()
        return super().apply(logits, *args)

    @staticmethod
    def forward(ctx, logits, tokens, ref_logprobs, beta=0.1, label_smoothing=0.0, ignore_index=-1, reduction="mean"):
        if ctx.needs_input_grad[2]:
            raise ValueError("ref_logprobs have no gradient; pass them detached")
        d = _desc(logits, tokens, ignore_index, reduction, 0, overwrite=True)
        dev, n, B = logits.device, tokens.numel(), tokens.shape[0]
        if B % 2 != 0:
            raise ValueError(f"answers come in pairs, got {B}")
        _check_tensor("ref_logprobs", ref_logprobs, (B,), _F32, dev)
        o = _lib.PreferenceOptions(float(beta), float(label_smoothing))
        # One allocation: the workspace (n float64), stats (2 n), weights (B), losses (B/2).
        room = torch.empty(4 * n + B + B // 2, dtype=torch.float32, device=dev)
        out = torch.empty((B // 2,) if reduction == "none" else (), dtype=torch.float32, device=dev)
        rewards = torch.empty((B,), dtype=torch.float32, device=dev)
        at = room.data_ptr()
        stats, weights = at + 8 * n, at + 16 * n
        losses, reduced = weights + 4 * B, out.data_ptr()
        if reduction == "none":
            losses, reduced = reduced, None
        _call(dev, _lib.lib().fc_preference_loss_fwd, ctypes.byref(d), ctypes.byref(o), logits.data_ptr(),
              tokens.data_ptr(), ref_logprobs.data_ptr(), losses, rewards.data_ptr(), None, stats, weights, reduced, at,
              8 * n)
        _save(ctx, d, logits, tokens, room)
        ctx.mark_non_differentiable(rewards)
        return out, rewards

    @staticmethod
    def backward(ctx, dout, _):
        logits, tokens, room = _as_saved(ctx.saved_tensors, _SAVED, ctx.saved_as, ctx.device)
        dout = _as_floats(dout)
        delta = _gradient_like(logits)
        at, n = room.data_ptr(), ctx.n
        _call(delta.device, _lib.lib().fc_preference_loss_bwd, ctypes.byref(ctx.desc), delta.data_ptr(), logits.data_ptr(),
              tokens.data_ptr(), at + 8 * n, at + 16 * n, dout.data_ptr())
        if torch.is_grad_enabled():
            delta = _OnceOnly.apply("the preference loss", delta, logits, dout)
        return (delta,) + (None,) * 6
