"""Losses over token log-probabilities for preference and policy tuning: the clipped policy loss with a KL term
(``molt_policy_loss_*``) and the loss over pairs of sequences (``molt_preference_loss_*``).  Forward and backward are
CUDA kernels; the reference, which trains on cross-entropy alone, has no counterpart."""
from __future__ import annotations

import ctypes
from typing import Any, NamedTuple, Optional

import torch

from molt_b200 import _native
from molt_b200.core.errors import CapabilityError

_REDUCTIONS = {"token": _native.REDUCE_TOKEN, "sequence": _native.REDUCE_SEQUENCE}
_KINDS = {"sigmoid": _native.PREFERENCE_SIGMOID, "hinge": _native.PREFERENCE_HINGE, "ipo": _native.PREFERENCE_IPO}


class PolicyLoss(NamedTuple):
    """Scalars on the device; only ``loss`` carries a gradient."""

    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class PreferenceLoss(NamedTuple):
    """``loss`` is a scalar that carries the gradient, the rewards are ``[pairs]`` and carry none."""

    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


def _check_logprobs(who: str, logprobs: torch.Tensor) -> None:
    if logprobs.device.type != "cuda":
        raise CapabilityError(f"{who} requires CUDA tensors")
    if logprobs.dtype != torch.float32:
        raise CapabilityError(f"{who} requires float32 log-probabilities")
    if logprobs.dim() != 2:
        raise ValueError("logprobs must be [sequences, tokens]")


def _check_like(name: str, tensor: torch.Tensor, logprobs: torch.Tensor, shape) -> None:
    if tensor.shape != shape or tensor.dtype != torch.float32 or tensor.device != logprobs.device:
        raise ValueError(f"{name} must be float32 of shape {tuple(shape)} on the device of logprobs")


def _check_mask(mask: Optional[torch.Tensor], logprobs: torch.Tensor) -> None:
    if mask is not None and (mask.shape != logprobs.shape or mask.dtype not in (torch.bool, torch.uint8)
                             or mask.device != logprobs.device):
        raise ValueError("mask must be bool or uint8 of the shape and on the device of logprobs")


def _rows(tensor: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The tensor, or a copy where its rows overlap or its tokens are not neighbours (rows may be one and the same)."""
    if tensor is None or tensor.dim() == 1 or tensor.is_contiguous():
        return tensor
    rows, width = tensor.shape
    neighbours = width <= 1 or tensor.stride(1) == 1
    apart = rows <= 1 or tensor.stride(0) == 0 or tensor.stride(0) >= width
    return tensor if neighbours and apart else tensor.contiguous()


def _row_stride(tensor: Optional[torch.Tensor]) -> int:
    if tensor is None or tensor.shape[0] <= 1:
        return 0
    return tensor.stride(0)


def _policy_forward(call, trained: bool):
    """Loss, ``[k, cut]`` and, for the backward pass, the gradients per token with the weights behind them."""
    lp, old, ref, advantages, mask, clip_low, clip_high, kl_coef, reduction = call
    lp, old, ref, mask, advantages = _rows(lp), _rows(old), _rows(ref), _rows(mask), _rows(advantages)
    batch, seq = lp.shape
    device = lp.device
    loss, stats = lp.new_empty(()), lp.new_empty(2)
    kept, unit, weight = None, None, None
    if trained:
        kept = lp.new_empty(batch * seq + batch + 1)
        unit = kept.data_ptr()
        weight = unit + 4 * batch * seq
    lib = _native.library()
    nbytes = lib.molt_policy_loss_workspace_bytes(batch, seq)
    scratch = _native.workspace(nbytes, device) if nbytes else None
    strides = (ctypes.c_int64 * 5)(*map(_row_stride, (lp, old, ref, advantages, mask)))
    with _native.on_device(device):
        _native.check(lib.molt_policy_loss_fwd(
            lp.data_ptr(), old.data_ptr(), _native.ptr(ref), advantages.data_ptr(), int(advantages.dim() == 2),
            _native.ptr(mask), strides, batch, seq, clip_low, clip_high, kl_coef, reduction, unit, weight, loss.data_ptr(),
            stats.data_ptr(), _native.ptr(scratch), nbytes, _native.stream_handle(device)))
    return loss, stats, kept


class _PolicyLossFunction(torch.autograd.Function):
    """Keeps one fp32 value per token and one per sequence for the backward pass; ``told`` receives the statistics."""

    @staticmethod
    def forward(ctx: Any, logprobs: torch.Tensor, call, told: list) -> torch.Tensor:
        loss, stats, kept = _policy_forward((logprobs, *call), True)
        told.append(stats)
        ctx.save_for_backward(kept)
        ctx.shape = logprobs.shape
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_loss: torch.Tensor):
        (kept,) = ctx.saved_tensors
        batch, seq = ctx.shape
        grad = kept.new_empty((batch, seq))
        unit = kept.data_ptr()
        with _native.on_device(kept.device):
            _native.check(_native.library().molt_policy_loss_bwd(unit, unit + 4 * batch * seq, grad_loss.data_ptr(), grad.data_ptr(),
                                                                 batch, seq, _native.stream_handle(kept.device)))
        return grad, None, None


def clipped_policy_loss(logprobs: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                        mask: Optional[torch.Tensor] = None, ref_logprobs: Optional[torch.Tensor] = None,
                        clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                        reduction: str = "token") -> PolicyLoss:
    """Mean over tokens of ``-min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl_coef k`` with
    ``r = exp(logprobs - old_logprobs)`` and ``k = exp(ref - logprobs) - (ref - logprobs) - 1``.

    ``logprobs``, ``old_logprobs`` and ``ref_logprobs`` are fp32 ``[sequences, tokens]``, ``advantages`` the same or
    ``[sequences]``.  Only tokens with a true ``mask`` count; what stands behind the mask is never used, NaN included.
    ``reduction="token"`` averages over all kept tokens, ``"sequence"`` over the sequences that keep one, of the mean over
    their kept tokens.  Without a kept token the loss and its gradient are zero.  Returns the loss, the mean ``k`` and the
    mean share of tokens whose gradient the clamp cut.  Only ``logprobs`` gets a gradient; a log-ratio on the clamp's
    border keeps its own."""
    _check_logprobs("clipped_policy_loss", logprobs)
    _check_like("old_logprobs", old_logprobs, logprobs, logprobs.shape)
    if ref_logprobs is not None:
        _check_like("ref_logprobs", ref_logprobs, logprobs, logprobs.shape)
    _check_like("advantages", advantages, logprobs, logprobs.shape if advantages.dim() == 2 else logprobs.shape[:1])
    _check_mask(mask, logprobs)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    _native.refuse_tangents("clipped_policy_loss", logprobs, old_logprobs, advantages, ref_logprobs)
    call = (old_logprobs, ref_logprobs, advantages, mask, float(clip_low), float(clip_high), float(kl_coef),
            _REDUCTIONS[reduction])
    if logprobs.requires_grad and torch.is_grad_enabled():
        told: list = []
        loss = _PolicyLossFunction.apply(logprobs, call, told)
        stats = told[0]
    else:
        loss, stats, _ = _policy_forward((logprobs, *call), False)
    return PolicyLoss(loss, stats[0], stats[1])


def _preference_forward(call, trained: bool):
    """Loss, rewards and, for the backward pass, the mask and the gradient of every sequence's tokens."""
    lp, ref, mask, beta, smoothing, kind, average = call
    lp, ref, mask = _rows(lp), _rows(ref), _rows(mask)
    sequences, seq = lp.shape
    pairs = sequences // 2
    device = lp.device
    loss, rewards = lp.new_empty(()), lp.new_empty((2, pairs))
    seq_grad = lp.new_empty(sequences) if trained else None
    lib = _native.library()
    nbytes = lib.molt_preference_loss_workspace_bytes(pairs, seq)
    scratch = _native.workspace(nbytes, device) if nbytes else None
    strides = (ctypes.c_int64 * 3)(*map(_row_stride, (lp, ref, mask)))
    with _native.on_device(device):
        _native.check(lib.molt_preference_loss_fwd(
            lp.data_ptr(), _native.ptr(ref), int(ref is not None and ref.dim() == 2), _native.ptr(mask), strides, pairs, seq,
            beta, smoothing, kind, average, _native.ptr(seq_grad), rewards.data_ptr(), loss.data_ptr(), _native.ptr(scratch), nbytes,
            _native.stream_handle(device)))
    return loss, rewards, mask, seq_grad


class _PreferenceLossFunction(torch.autograd.Function):
    """Keeps the mask and one fp32 value per sequence for the backward pass; ``told`` receives the rewards."""

    @staticmethod
    def forward(ctx: Any, logprobs: torch.Tensor, call, told: list) -> torch.Tensor:
        loss, rewards, mask, seq_grad = _preference_forward((logprobs, *call), True)
        told.append(rewards)
        ctx.save_for_backward(mask, seq_grad)
        ctx.shape = logprobs.shape
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_loss: torch.Tensor):
        mask, seq_grad = ctx.saved_tensors
        sequences, seq = ctx.shape
        grad = seq_grad.new_empty((sequences, seq))
        with _native.on_device(grad.device):
            _native.check(_native.library().molt_preference_loss_bwd(
                _native.ptr(mask), _row_stride(mask), seq_grad.data_ptr(), grad_loss.data_ptr(), grad.data_ptr(), sequences // 2, seq,
                _native.stream_handle(grad.device)))
        return grad, None, None


def preference_loss(logprobs: torch.Tensor, ref_logprobs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                    beta: float = 0.1, label_smoothing: float = 0.0, kind: str = "sigmoid",
                    average: bool = False) -> PreferenceLoss:
    """Loss over pairs of sequences from their token log-probabilities (fp32 ``[2 * pairs, tokens]``: the chosen sequences,
    then the rejected ones in the same order).

    With ``s`` the sum over a sequence's kept tokens of ``logprobs - ref_logprobs`` (``average``: their mean) and
    ``h = s_chosen - s_rejected``, the mean over pairs of ``-(1 - e) ln sig(beta h) - e ln sig(-beta h)`` for ``"sigmoid"``
    (``e`` the label smoothing), ``max(0, 1 - beta h)`` for ``"hinge"``, ``(h - 1 / (2 beta))^2`` for ``"ipo"``.
    ``ref_logprobs`` is ``[2 * pairs, tokens]``, or ``[2 * pairs]`` sums (means with ``average``) kept from an earlier pass, or
    None (zero).  What stands behind the mask is never used; a sequence that keeps no token has ``s = 0``.  The rewards
    are ``beta s``.  Only ``logprobs`` gets a gradient."""
    _check_logprobs("preference_loss", logprobs)
    if logprobs.shape[0] == 0 or logprobs.shape[0] % 2:
        raise ValueError("logprobs must hold the chosen sequences and then as many rejected ones")
    if ref_logprobs is not None:
        _check_like("ref_logprobs", ref_logprobs, logprobs,
                    logprobs.shape if ref_logprobs.dim() == 2 else logprobs.shape[:1])
    _check_mask(mask, logprobs)
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)}")
    _native.refuse_tangents("preference_loss", logprobs, ref_logprobs)
    call = (ref_logprobs, mask, float(beta), float(label_smoothing), _KINDS[kind], int(bool(average)))
    if logprobs.requires_grad and torch.is_grad_enabled():
        told: list = []
        loss = _PreferenceLossFunction.apply(logprobs, call, told)
        rewards = told[0]
    else:
        loss, rewards, _, _ = _preference_forward((logprobs, *call), False)
    return PreferenceLoss(loss, rewards[0], rewards[1])
