"""Global gradient norm over many tensors, and clipping (``molt_grad_norm``, ``molt_clip_grads``): what stands between a
backward pass and the optimizer step.  Nothing is read back to the host."""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from molt_b200 import _native
from molt_b200.core.errors import CapabilityError

_NORMS = {2.0: _native.NORM_L2, float("inf"): _native.NORM_MAX}

Grads = Union[torch.Tensor, Sequence[torch.Tensor]]


def _dense(tensor: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in whatever order."""
    expect = 1
    for extent, stride in sorted(zip(tensor.shape, tensor.stride()), key=lambda p: (p[1], p[0])):
        if extent != 1:
            if stride != expect:
                return False
            expect *= extent
    return True


def _checked(name: str, tensors: Grads) -> Tuple[Tuple[torch.Tensor, ...], bool]:
    """The tensors as a tuple, and whether all of them are contiguous; raises for one that has gaps or repeats elements."""
    tensors = (tensors,) if isinstance(tensors, torch.Tensor) else tuple(tensors)
    if not tensors:
        raise ValueError(f"{name}: at least one tensor is needed")
    contiguous = all(map(torch.Tensor.is_contiguous, tensors))
    if not contiguous and not all(t.numel() == 0 or _dense(t) for t in tensors):
        raise ValueError(f"{name}: every tensor must fill its memory (no gaps, no repeated elements)")
    return tensors, contiguous


def _norm_kind(norm_type: float) -> int:
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise CapabilityError("the gradient norm is 2 or inf")
    return kind


def _check_device(grads: Tuple[torch.Tensor, ...]) -> None:
    if grads[0].device.type != "cuda" or len(set(map(torch.Tensor.get_device, grads))) != 1:
        if any(t.device.type != "cuda" for t in grads):
            raise CapabilityError("gradient norms require CUDA tensors")
        raise ValueError("all gradients must be on one device")


def _launch(grads: Tuple[torch.Tensor, ...], outs: Optional[Tuple[torch.Tensor, ...]], kind: int, max_norm: float) -> torch.Tensor:
    _check_device(grads)
    _native.refuse_tangents("the gradient norm", *grads)
    items, device, count = _native.grad_items(grads, outs), grads[0].device, len(grads)
    lib = _native.library()
    scratch = _native.workspace(lib.molt_grad_norm_workspace_bytes(count), device)
    result = torch.empty(2, dtype=torch.float32, device=device)
    with _native.on_device(device):
        if outs is None:
            _native.check(lib.molt_grad_norm(items.buffer_info()[0], count, kind, 1.0, max_norm, result.data_ptr(),
                                             scratch.data_ptr(), scratch.numel(), _native.stream_handle(device)))
        else:
            _native.check(lib.molt_clip_grads(items.buffer_info()[0], count, kind, max_norm, result.data_ptr(),
                                              scratch.data_ptr(), scratch.numel(), _native.stream_handle(device)))
    return result[0]


def global_grad_norm(grads: Grads, norm_type: float = 2.0) -> torch.Tensor:
    """Norm of all elements of ``grads`` (one tensor or a sequence; bf16 and fp32 may be mixed) as an fp32 scalar on the
    device: the square root of the sum of squares (``norm_type`` 2) or the largest magnitude (``inf``).  Squares of any finite
    gradient are held; a norm beyond fp32's range is reported as fp32's largest value.  A NaN gives NaN, and an infinity
    infinity.  Equal lists of equal alignment (to 16 bytes) give equal bits.  Nothing is recorded for autograd."""
    grads, _ = _checked("grads", grads)
    return _launch(grads, None, _norm_kind(norm_type), float("inf"))


def clip_grad_norm(grads: Grads, max_norm: float, norm_type: float = 2.0, out: Optional[Grads] = None) -> torch.Tensor:
    """Scale ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and return their :func:`global_grad_norm` before that.  The
    factor is formed from the norm in 64 bits, so finite gradients are clipped rightly where their norm leaves fp32 too.

    In place, or into ``out``: tensors of the same dtypes and sizes that lie in memory as ``grads`` do (of contiguous ones the
    shapes may differ).  An output may be its own gradient but must not overlap another tensor of the call.  One tensor must
    not stand in the list twice.  Nothing is recorded for autograd."""
    grads, plain = _checked("grads", grads)
    kind = _norm_kind(norm_type)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    outs = grads
    if out is not None and out is not grads:
        outs, plain_outs = _checked("out", out)
        numel, get_device = torch.Tensor.numel, torch.Tensor.get_device   # whole lists at a time: there may be hundreds
        if (list(map(numel, outs)) != list(map(numel, grads)) or list(map(get_device, outs)) != list(map(get_device, grads))
                or [t.dtype for t in outs] != [t.dtype for t in grads]):
            raise ValueError("out must match grads in number, size, dtype and device")
        if not (plain and plain_outs) and any(o.shape != g.shape or o.stride() != g.stride() for o, g in zip(outs, grads)
                                              if not (o.is_contiguous() and g.is_contiguous())):
            raise ValueError("out must lie in memory as grads do")
    norm = _launch(grads, outs, kind, float(max_norm))
    torch.autograd.graph.increment_version(outs)
    return norm
