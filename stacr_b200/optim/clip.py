"""Global gradient norm and clipping by it, over all parameters in two kernel launches (``csrc/grad_clip.cu``)."""

from __future__ import annotations

from array import array
from typing import Iterable

import torch

_KERNEL_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _parameters(parameters) -> list[torch.Tensor]:
    return [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _kernel_table(grads):
    """``(pointers, sizes, type codes)`` of the distinct gradients, or ``None`` where the kernel does not apply."""
    if not grads or not grads[0].is_cuda:
        return None
    device = grads[0].get_device()
    seen = {}
    for g in grads:
        code = _KERNEL_DTYPES.get(g.dtype)
        if code is None or type(g) is not torch.Tensor or g.layout is not torch.strided or g.get_device() != device or not (g.is_contiguous() or _dense(g)):
            return None
        n = g.numel()
        if n:
            seen[g.data_ptr(), n, code] = None
    end = 0
    for start, n, code in sorted(seen):
        if start < end:
            raise ValueError("two gradients overlap in memory: clipping would scale the shared elements twice")
        end = start + n * (4 if code == 2 else 2)
    return [*zip(*seen)] if seen else ((), (), ())


def _run(grads, table, max_norm: float | None) -> torch.Tensor:
    from ..ops import _lib

    ptrs, sizes, codes = table
    n = len(ptrs)
    if not n:
        return torch.zeros((), dtype=torch.float32, device=grads[0].device)
    with _lib.on_device(grads[0]):
        sms, stream = _lib.place(grads[0])
        norm = grads[0].new_empty((), dtype=torch.float32)
        partial = norm.new_empty(_lib.entry("sb_clip_partials", "ii")(n, sms), dtype=torch.float64)
        ptrs, sizes, codes = array("Q", ptrs), array("q", sizes), array("B", codes)
        rc = _lib.entry("sb_grad_clip", "pppippdiip")(ptrs.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], n, partial.data_ptr(), norm.data_ptr(),
                                                     0.0 if max_norm is None else max_norm, max_norm is not None, sms, stream)
    _lib.check_rc(rc, "sb_grad_clip")
    groups = -(-n // _lib.entry("sb_clip_tensors_per_launch", "")())
    _lib.count(groups + (1 if max_norm is None else groups))
    return norm


def grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """2-norm of all gradients together as a device scalar, without waiting for the device.  A gradient that occurs twice counts once."""
    grads = [p.grad for p in _parameters(parameters) if p.grad is not None]
    table = _kernel_table(grads)
    if table is None:
        return torch.nn.utils.get_total_norm(list({id(g): g for g in grads}.values()))
    return _run(grads, table, None)


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """Scale all gradients in place by ``min(1, max_norm / (norm + 1e-6))`` and return their norm from before, as a device scalar.

    Dense bf16, fp16 and fp32 gradients on one GPU take the kernels, which sum the 2-norm beyond fp32's range and decide about the
    scaling on the device, so the host does not wait (``error_if_nonfinite`` does, and raises before anything is scaled) and the
    call can be captured into a CUDA graph.  A gradient that occurs twice counts and is scaled once; gradients that overlap in part
    are refused.  Everything else (other norms, other layouts or devices, sharded tensors) goes to the framework's function, with
    ``foreach``.
    """
    max_norm, norm_type = float(max_norm), float(norm_type)
    params = _parameters(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    table = _kernel_table(grads) if norm_type == 2.0 else None
    if table is None:
        return torch.nn.utils.clip_grad_norm_(params, max_norm, norm_type, error_if_nonfinite, foreach)
    if error_if_nonfinite:
        norm = _run(grads, table, None)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: they were left unscaled (error_if_nonfinite)")
    norm = _run(grads, table, max_norm)
    torch.autograd.graph.increment_version(grads)
    return norm
