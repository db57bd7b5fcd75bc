"""The kernels behind ``nn_ops.gated_linear`` (``csrc/gated_gemm.cu``) on contiguous bf16 matrices: ``x [M, K]``, weights ``[F, K]``,
results ``[M, F]``; biases fp32 or ``None``; ``K`` and ``F`` multiples of 8."""

from __future__ import annotations

import torch

from . import _lib
from .nn_kernels import ACTIVATION_CODE


def _ptr(t):
    return None if t is None else t.data_ptr()


def forward(x, wg, wu, bg, bu, activation: str, keep: bool):
    """``(h, kept)``: with ``keep`` a byte buffer with the backward's two factors, 16 bits of each value ``[2, M, F]`` and behind them 8
    ``[2, M, F padded to 16]``."""
    m, k = x.shape
    f = wg.shape[0]
    h = x.new_empty((m, f))
    kept = hi = lo = None
    if keep:
        kept = x.new_empty(4 * m * f + 2 * m * ((f + 15) // 16 * 16), dtype=torch.uint8)
        hi = kept.data_ptr()
        lo = hi + 4 * m * f
    sms, stream = _lib.place(x)
    rc = _lib.entry("sb_gated_forward", "ppppppppiiiiipp")(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), h.data_ptr(), hi, lo, m, k, f,
                                                         ACTIVATION_CODE[activation], sms, _lib.status_word(x.device).data_ptr(), stream)
    _lib.check_rc(rc, "sb_gated_forward")
    _lib.count(1)
    return h, kept


def backward(dh, x, wg, wu, bg, bu, activation: str, kept, need_dx: bool, out_gate, out_up):
    """``(d, dx)``: ``d [2, M, F]`` holds dgate and dup, from what :func:`forward` kept or from the projections formed again, and
    ``dx = dgate Wg + dup Wu``.  ``dgate^T x`` and ``dup^T x`` go to ``out_gate`` and ``out_up``, fp32 or bf16 ``[F, K]`` or ``None``."""
    m, k = x.shape
    f = dh.shape[1]
    d = x.new_empty((2, m, f))
    dx = torch.empty_like(x) if need_dx else None
    hi = lo = None
    if kept is not None:
        hi = kept.data_ptr()
        lo = hi + 4 * m * f
    sms, stream = _lib.place(x)
    size = _lib.entry("sb_gated_partial_bytes", "iiiiii", "l")(m, k, f, need_dx, int(out_gate is not None) + int(out_up is not None), sms)
    partial = x.new_empty(size, dtype=torch.uint8) if size else None       # sums of split reductions
    rc = _lib.entry("sb_gated_backward", "pppppppppppp" + "pl" + "iiiiiii" + "pp")(
        dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), hi, lo, d.data_ptr(), _ptr(dx), _ptr(out_gate), _ptr(out_up),
        _ptr(partial), size, out_gate is not None and out_gate.dtype == torch.float32, out_up is not None and out_up.dtype == torch.float32, m, k, f,
        ACTIVATION_CODE[activation], sms, _lib.status_word(x.device).data_ptr(), stream)
    _lib.check_rc(rc, "sb_gated_backward")
    _lib.count(1 + int(need_dx) + int(out_gate is not None or out_up is not None))
    return d, dx
