"""Log-probabilities of given tokens from logits (``molt_token_logprob_*``): what preference and policy losses, and the
scoring of sampled text, are made of.  The logits' softmax is never stored; the reference has no counterpart (it trains
on cross-entropy alone, reference kernels/frozen_linear_cross_entropy.py:181-236)."""
from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from molt_b200 import _native
from molt_b200.core.errors import CapabilityError

_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float32: _native.DTYPE_F32}


def _check(logits: torch.Tensor, token_ids: torch.Tensor) -> int:
    if logits.device.type != "cuda":
        raise CapabilityError("token log-probabilities require CUDA tensors")
    if logits.dtype not in _DTYPES:
        raise CapabilityError("token log-probabilities support bfloat16 and float32 logits")
    if logits.dim() < 1 or logits.shape[:-1] != token_ids.shape or logits.shape[-1] == 0:
        raise ValueError("logits must be [..., vocab] with token_ids of the leading shape")
    if token_ids.dtype != torch.int64 or token_ids.device != logits.device:
        raise ValueError("token_ids must be int64 on the logits' device")
    return _DTYPES[logits.dtype]


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """``[rows, vocab]`` with neighbouring columns: a view where the strides allow it, else a copy."""
    if logits.dim() == 2 and logits.is_contiguous():
        return logits
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if (rows.shape[1] != 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and 0 < rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    return rows


def _stride(rows: torch.Tensor) -> int:
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _forward(rows: torch.Tensor, ids: torch.Tensor, temperature: float, stats: Optional[torch.Tensor]) -> torch.Tensor:
    device = rows.device
    logprobs = torch.empty(ids.shape, dtype=torch.float32, device=device)
    with _native.on_device(device):
        _native.check(_native.library().molt_token_logprob_fwd(
            rows.data_ptr(), _DTYPES[rows.dtype], _stride(rows), ids.data_ptr(), temperature, logprobs.data_ptr(),
            _native.ptr(stats), rows.shape[0], rows.shape[1], _native.stream_handle(device)))
    return logprobs


class _TokenLogprobs(torch.autograd.Function):
    """Saves the logits (by reference), the ids and two floats per row."""

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, token_ids: torch.Tensor, temperature: float) -> torch.Tensor:
        rows, ids = _rows(logits), token_ids.contiguous()
        stats = torch.empty((rows.shape[0], 2), dtype=torch.float32, device=rows.device)
        ctx.save_for_backward(rows, ids, stats)
        ctx.shape, ctx.temperature = logits.shape, temperature
        return _forward(rows, ids, temperature, stats)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: torch.Tensor):
        rows, ids, stats = ctx.saved_tensors
        grad_output = grad_output.contiguous()
        grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        with _native.on_device(rows.device):
            _native.check(_native.library().molt_token_logprob_bwd(
                rows.data_ptr(), _DTYPES[rows.dtype], _stride(rows), ids.data_ptr(), stats.data_ptr(), grad_output.data_ptr(),
                ctx.temperature, grad.data_ptr(), grad.shape[1], rows.shape[0], rows.shape[1],
                _native.stream_handle(rows.device)))
        return grad.reshape(ctx.shape), None, None


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """``log_softmax(logits / temperature)[..., token_ids]`` in fp32, differentiable with respect to the logits.

    ``logits`` is ``[..., vocab]`` in bf16 or fp32 (any row stride), ``token_ids`` int64 of the leading shape.  A token id
    outside ``[0, vocab)`` (an ignore index such as -100) gives 0 and no gradient, whatever its row holds.  Logits of -inf
    have probability zero; a row without a finite logit, or with a NaN or +inf, gives NaN."""
    _check(logits, token_ids)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogprobs.apply(logits, token_ids, float(temperature))
    return _forward(_rows(logits), token_ids.contiguous(), float(temperature), None)


def token_logprobs_with_grad(logits: torch.Tensor, token_ids: torch.Tensor, weight: Optional[torch.Tensor] = None,
                             temperature: float = 1.0, out: Optional[torch.Tensor] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(logprobs, grad)`` in one pass over the logits: the log-probabilities of :func:`token_logprobs` (to rounding) and
    ``grad[..., v] = weight * d logprob / d logits[..., v]`` (``weight`` None: 1), rounded once to the logits' type.

    For callers that differentiate by hand, such as a head whose logits are not kept: ``out`` receives the gradient and may
    be ``logits`` itself, which it then overwrites (it must not overlap them in any other way).  Nothing is recorded for
    autograd."""
    dtype = _check(logits, token_ids)
    rows, ids = _rows(logits.detach()), token_ids.contiguous()
    if weight is not None:
        if weight.shape != token_ids.shape or weight.dtype != torch.float32 or weight.device != logits.device:
            raise ValueError("weight must be float32 of the shape of token_ids on the logits' device")
        weight = weight.detach().contiguous()
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, dtype and device")
    elif out.requires_grad:
        raise ValueError("out must not require a gradient")
    target = out
    if out.dim() != 2:
        try:
            target = out.view(-1, out.shape[-1])
        except RuntimeError as exc:
            raise ValueError("out must be a tensor of rows with one stride") from exc
    if target.shape[1] != 1 and target.stride(1) != 1:
        raise ValueError("out must have neighbouring columns")
    logprobs = torch.empty(token_ids.shape, dtype=torch.float32, device=logits.device)
    with _native.on_device(logits.device):
        _native.check(_native.library().molt_token_logprob_grad(
            rows.data_ptr(), dtype, _stride(rows), ids.data_ptr(), _native.ptr(weight), float(temperature), logprobs.data_ptr(),
            target.data_ptr(), _stride(target), rows.shape[0], rows.shape[1], _native.stream_handle(logits.device)))
    torch.autograd.graph.increment_version(out)
    return logprobs, out
