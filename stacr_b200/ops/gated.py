"""The kernels behind ``nn_ops.gated_linear`` (``csrc/gated_gemm.cu``) on contiguous bf16 matrices: ``x [M, K]``, weights ``[F, K]``,
results ``[M, F]``; biases fp32 or ``None``; ``K`` and ``F`` multiples of 8."""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .nn_kernels import ACTIVATION_CODE

_TYPED = None


def _typed_lib():
    """The kernel library with the argument types of these entry points declared: plain Python numbers then convert by themselves."""
    global _TYPED
    if _TYPED is None:
        lib = _lib.load()
        vp, ci = ctypes.c_void_p, ctypes.c_int
        for name, args in {"sb_gated_forward": [vp] * 10 + [ci] * 5 + [vp] * 2, "sb_gated_recompute": [vp] * 8 + [ci] * 5 + [vp] * 2,
                           "sb_gated_factors": [vp] * 7 + [ci] * 3 + [vp], "sb_gated_input_grad": [vp] * 5 + [ci] * 4 + [vp] * 2,
                           "sb_gated_weight_grads": [vp] * 5 + [ci] * 6 + [vp] * 2}.items():
            getattr(lib, name).argtypes, getattr(lib, name).restype = args, ci
        _TYPED = lib
    return _TYPED


def _ptr(t):
    return None if t is None else t.data_ptr()


def _common(t):
    return _lib.sm_count(t.device), _lib.status_word(t.device).data_ptr(), _lib.stream_ptr()


def _done(rc: int, name: str) -> None:
    _lib.check_rc(rc, name)
    _lib.count(1)


def forward(x, wg, wu, bg, bu, activation: str, keep: bool):
    """``(h, kept)``: with ``keep`` the backward's two factors as ``(a_hi, a_lo, b_hi, b_lo)``, 16 and 8 bits of each value."""
    m, k = x.shape
    f = wg.shape[0]
    h = torch.empty(m, f, dtype=torch.bfloat16, device=x.device)
    kept = None
    if keep:
        hi, lo = torch.empty(2, m, f, dtype=torch.int16, device=x.device), torch.empty(2, m, -(-f // 16) * 16, dtype=torch.uint8, device=x.device)
        kept = hi[0], lo[0], hi[1], lo[1]      # every part starts on 16 bytes: f is a multiple of 8
    a_hi, a_lo, b_hi, b_lo = (t.data_ptr() for t in kept) if keep else (None,) * 4
    rc = _typed_lib().sb_gated_forward(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), h.data_ptr(), a_hi, a_lo, b_hi, b_lo, m, k, f,
                                       ACTIVATION_CODE[activation], *_common(x))
    _done(rc, "sb_gated_forward")
    return h, kept


def backward_kept(dh, a_hi, a_lo, b_hi, b_lo):
    """``(dgate, dup)`` from what :func:`forward` kept."""
    m, f = dh.shape
    dg, du = torch.empty_like(dh), torch.empty_like(dh)
    rc = _typed_lib().sb_gated_factors(dh.data_ptr(), a_hi.data_ptr(), a_lo.data_ptr(), b_hi.data_ptr(), b_lo.data_ptr(), dg.data_ptr(), du.data_ptr(), m, f,
                                       _lib.sm_count(dh.device), _lib.stream_ptr())
    _done(rc, "sb_gated_factors")
    return dg, du


def backward_recomputed(dh, x, wg, wu, bg, bu, activation: str):
    """``(dgate, dup)`` with the projections formed again."""
    m, k = x.shape
    dg, du = torch.empty_like(dh), torch.empty_like(dh)
    rc = _typed_lib().sb_gated_recompute(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), dh.data_ptr(), dg.data_ptr(), du.data_ptr(), m, k,
                                         wg.shape[0], ACTIVATION_CODE[activation], *_common(x))
    _done(rc, "sb_gated_recompute")
    return dg, du


def input_gradient(dg, du, wg, wu):
    """``dgate Wg + dup Wu`` in bf16, summed in fp32."""
    m, f = dg.shape
    k = wg.shape[1]
    dx = torch.empty(m, k, dtype=torch.bfloat16, device=dg.device)
    rc = _typed_lib().sb_gated_input_grad(dg.data_ptr(), du.data_ptr(), wg.data_ptr(), wu.data_ptr(), dx.data_ptr(), m, k, f, *_common(dg))
    _done(rc, "sb_gated_input_grad")
    return dx


def weight_gradients(dg, du, x, gate_dtype, up_dtype, slots, need_gate: bool, need_up: bool):
    """``(dgate^T x, dup^T x)``, fp32 into a slot or for an fp32 weight, bf16 otherwise; ``None`` for one that is not needed."""
    m, k = x.shape
    out = []
    for dtype, slot, need in ((gate_dtype, slots[0], need_gate), (up_dtype, slots[1], need_up)):
        kind = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        out.append(None if not need else slot if slot is not None else torch.empty(dg.shape[1], k, dtype=kind, device=x.device))
    rc = _typed_lib().sb_gated_weight_grads(dg.data_ptr(), du.data_ptr(), x.data_ptr(), _ptr(out[0]), _ptr(out[1]),
                                            *(int(t is not None and t.dtype == torch.float32) for t in out), m, k, dg.shape[1], *_common(x))
    _done(rc, "sb_gated_weight_grads")
    return out
