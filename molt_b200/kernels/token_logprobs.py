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


def _read_where_it_is(logits: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, int, int]]:
    """The tensor, or a copy where it has to be one, and how its rows lie: (row stride, rows per group, group stride).  Rows that
    two strides describe, such as those of ``logits[:, :-1]``, are read where they are."""
    vocab = logits.shape[-1]
    if logits.is_contiguous():
        return logits, (vocab, 0, 0)
    levels: list = []   # (extent, stride) of the leading dimensions from the last to the first, joined where they follow on
    for extent, stride in zip(reversed(logits.shape[:-1]), reversed(logits.stride()[:-1])):
        if extent == 1:
            continue
        if levels and stride == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * extent, levels[-1][1])
        else:
            levels.append((extent, stride))
    if len(levels) > 2 or (vocab != 1 and logits.stride(-1) != 1) or any(0 < stride < vocab for _, stride in levels):
        return logits.contiguous(), (vocab, 0, 0)
    levels += [(0, vocab)] * (2 - len(levels))
    (group_rows, row_stride), (_, group_stride) = levels
    return logits, (row_stride, group_rows, group_stride)


def _stride(rows: torch.Tensor) -> int:
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _forward(rows: torch.Tensor, layout: Tuple[int, int, int], ids: torch.Tensor, temperature: float,
             stats: Optional[torch.Tensor]) -> torch.Tensor:
    device = rows.device
    logprobs = torch.empty(ids.shape, dtype=torch.float32, device=device)
    with _native.on_device(device):
        _native.check(_native.library().molt_token_logprob_fwd(
            rows.data_ptr(), _DTYPES[rows.dtype], *layout, ids.data_ptr(), temperature, logprobs.data_ptr(), _native.ptr(stats),
            ids.numel(), rows.shape[-1], _native.stream_handle(device)))
    return logprobs


class _TokenLogprobs(torch.autograd.Function):
    """Saves the logits (by reference), the ids and two floats per row."""

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, token_ids: torch.Tensor, temperature: float) -> torch.Tensor:
        (rows, layout), ids = _read_where_it_is(logits), token_ids.contiguous()
        stats = torch.empty((ids.numel(), 2), dtype=torch.float32, device=rows.device)
        ctx.save_for_backward(rows, ids, stats)
        ctx.layout, ctx.temperature = layout, temperature
        return _forward(rows, layout, ids, temperature, stats)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: torch.Tensor):
        rows, ids, stats = ctx.saved_tensors
        grad_output = grad_output.contiguous()
        grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        with _native.on_device(rows.device):
            _native.check(_native.library().molt_token_logprob_bwd(
                rows.data_ptr(), _DTYPES[rows.dtype], *ctx.layout, ids.data_ptr(), stats.data_ptr(), grad_output.data_ptr(),
                ctx.temperature, grad.data_ptr(), grad.shape[-1], ids.numel(), grad.shape[-1],
                _native.stream_handle(rows.device)))
        return grad, None, None


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """``log_softmax(logits / temperature)[..., token_ids]`` in fp32, differentiable with respect to the logits.

    ``logits`` is ``[..., vocab]`` in bf16 or fp32 (a slice such as ``logits[:, :-1]`` is read where it is), ``token_ids`` int64 of the leading shape.  A token id
    outside ``[0, vocab)`` (an ignore index such as -100) gives 0 and no gradient, whatever its row holds.  Logits of -inf
    have probability zero; a row without a finite logit, or with a NaN or +inf, gives NaN."""
    _check(logits, token_ids)
    _native.refuse_tangents("token_logprobs", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogprobs.apply(logits, token_ids, float(temperature))
    return _forward(*_read_where_it_is(logits), token_ids.contiguous(), float(temperature), None)


def token_logprobs_with_grad(logits: torch.Tensor, token_ids: torch.Tensor, weight: Optional[torch.Tensor] = None,
                             temperature: float = 1.0, out: Optional[torch.Tensor] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(logprobs, grad)`` in one pass over the logits: the log-probabilities of :func:`token_logprobs` (to rounding) and
    ``grad[..., v] = weight * d logprob / d logits[..., v]`` (``weight`` None: 1), rounded once to the logits' type.

    For callers that differentiate by hand, such as a head whose logits are not kept: ``out`` receives the gradient and may
    be ``logits`` itself, which it then overwrites (it must not overlap them in any other way).  Nothing is recorded for
    autograd."""
    dtype = _check(logits, token_ids)
    _native.refuse_tangents("token_logprobs_with_grad", logits, weight, out)
    (rows, layout), ids = _read_where_it_is(logits.detach()), token_ids.contiguous()
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
            rows.data_ptr(), dtype, *layout, ids.data_ptr(), _native.ptr(weight), float(temperature), logprobs.data_ptr(),
            target.data_ptr(), _stride(target), ids.numel(), rows.shape[-1], _native.stream_handle(logits.device)))
    torch.autograd.graph.increment_version(out)
    return logprobs, out
