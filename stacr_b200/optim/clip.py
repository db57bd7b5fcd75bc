"""Global gradient norm and clipping by it, over all parameters in two kernel launches (``csrc/grad_clip.cu``)."""

from __future__ import annotations

import ctypes
from typing import Iterable

import numpy as np
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
    device = grads[0].device if grads else None
    if device is None or device.type != "cuda":
        return None
    for g in grads:
        if type(g) is not torch.Tensor or g.device != device or g.dtype not in _KERNEL_DTYPES or g.layout != torch.strided or not _dense(g):
            return None
    seen = {}
    for g in grads:
        if g.numel():
            seen.setdefault((g.data_ptr(), g.numel(), g.dtype), g)
    ptrs = np.array([key[0] for key in seen], dtype=np.uint64)
    sizes = np.array([key[1] for key in seen], dtype=np.int64)
    codes = np.array([_KERNEL_DTYPES[key[2]] for key in seen], dtype=np.uint8)
    order = np.argsort(ptrs, kind="stable")
    ends = ptrs + sizes.astype(np.uint64) * np.where(codes == 2, 4, 2).astype(np.uint64)
    if (ends[order][:-1] > ptrs[order][1:]).any():
        raise ValueError("two gradients overlap in memory: clipping would scale the shared elements twice")
    return ptrs, sizes, codes


def _run(grads, table, max_norm: float | None) -> torch.Tensor:
    from ..ops import _lib

    ptrs, sizes, codes = table
    device = grads[0].device
    if not len(ptrs):
        return torch.zeros((), dtype=torch.float32, device=device)
    lib = _lib.load()
    with _lib.on_device(grads[0]):
        sms = _lib.sm_count(device)
        norm = torch.empty((), dtype=torch.float32, device=device)
        partial = torch.empty(lib.sb_clip_partials(ctypes.c_int(len(ptrs)), ctypes.c_int(sms)), dtype=torch.float64, device=device)
        rc = lib.sb_grad_clip(ctypes.c_void_p(ptrs.ctypes.data), ctypes.c_void_p(sizes.ctypes.data), ctypes.c_void_p(codes.ctypes.data),
                              ctypes.c_int(len(ptrs)), _lib.ptr(partial), _lib.ptr(norm), ctypes.c_double(0.0 if max_norm is None else max_norm),
                              ctypes.c_int(int(max_norm is not None)), ctypes.c_int(sms), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_grad_clip")
    groups = -(-len(ptrs) // lib.sb_clip_tensors_per_launch())
    _lib.count(groups + (1 if max_norm is None else groups))
    return norm


@torch.no_grad()
def grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """2-norm of all gradients together as a device scalar, without waiting for the device.  A gradient that occurs twice counts once."""
    grads = [p.grad for p in _parameters(parameters) if p.grad is not None]
    table = _kernel_table(grads)
    if table is None:
        return torch.nn.utils.get_total_norm(list({id(g): g for g in grads}.values()))
    return _run(grads, table, None)


@torch.no_grad()
def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale all gradients in place by ``min(1, max_norm / (norm + 1e-6))`` and return their norm from before, as a device scalar.

    The call of ``torch.nn.utils.clip_grad_norm_``.  Dense bf16, fp16 and fp32 gradients on one GPU take the kernels, which sum the
    2-norm beyond fp32's range and decide about the scaling on the device, so the host does not wait (``error_if_nonfinite``
    does, and raises before anything is scaled) and the call can be captured into a CUDA graph.  A gradient that occurs
    twice counts and is scaled once; gradients that overlap in part are refused.  Everything else (other norms, other layouts or
    devices, sharded tensors) goes to the framework's function.
    """
    max_norm, norm_type = float(max_norm), float(norm_type)
    params = _parameters(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    table = _kernel_table(grads) if norm_type == 2.0 else None
    if table is None:
        return torch.nn.utils.clip_grad_norm_(params, max_norm, norm_type, error_if_nonfinite)
    if error_if_nonfinite:
        norm = _run(grads, table, None)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot be clipped. "
                               "To disable this error and scale the gradients by the non-finite norm anyway, set `error_if_nonfinite=False`")
    norm = _run(grads, table, max_norm)
    for g in grads:
        torch.autograd.graph.increment_version(g)
    return norm
