"""ctypes entry points for ``csrc/nn_kernels.cu`` (LayerNorm, GELU, cross-entropy, casts), ``csrc/gated.cu`` and ``csrc/rotary.cu``."""

from __future__ import annotations

import ctypes

import torch

from . import _lib

c_int, c_ll, c_float = ctypes.c_int, ctypes.c_longlong, ctypes.c_float


def _f32(t):
    return None if t is None else t.detach().float().contiguous()


def layernorm_fwd(x2d: torch.Tensor, weight, bias, eps: float):
    rows, n = x2d.shape
    y = torch.empty_like(x2d)
    mean = torch.empty(rows, dtype=torch.float32, device=x2d.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x2d.device)
    rc = _lib.load().sb_layernorm_fwd(_lib.ptr(x2d), _lib.ptr(_f32(weight)), _lib.ptr(_f32(bias)), c_int(rows), c_int(n), c_float(eps),
                                      _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_layernorm_fwd")
    _lib.count(1)
    return y, mean, rstd


def layernorm_bwd(dy2d, x2d, weight, mean, rstd):
    rows, n = x2d.shape
    dx = torch.empty_like(x2d)
    dwb = torch.zeros(2, n, dtype=torch.float32, device=x2d.device)
    rc = _lib.load().sb_layernorm_bwd(_lib.ptr(dy2d), _lib.ptr(x2d), _lib.ptr(_f32(weight)), _lib.ptr(mean), _lib.ptr(rstd), c_int(rows),
                                      c_int(n), _lib.ptr(dx), _lib.ptr(dwb[0]), _lib.ptr(dwb[1]), c_int(_lib.sm_count(x2d.device)),
                                      _lib.stream_ptr())
    _lib.check_rc(rc, "sb_layernorm_bwd")
    _lib.count(2)
    return dx, dwb[0], dwb[1]


def layernorm_fwd2(x2d: torch.Tensor, w1, b1, w2, b2, eps: float):
    """Two affine outputs of one normalisation of ``x2d`` (one read of the input, shared statistics)."""
    rows, n = x2d.shape
    y1, y2 = torch.empty_like(x2d), torch.empty_like(x2d)
    mean = torch.empty(rows, dtype=torch.float32, device=x2d.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x2d.device)
    rc = _lib.load().sb_layernorm_fwd2(_lib.ptr(x2d), _lib.ptr(_f32(w1)), _lib.ptr(_f32(b1)), _lib.ptr(_f32(w2)), _lib.ptr(_f32(b2)), c_int(rows),
                                       c_int(n), c_float(eps), _lib.ptr(y1), _lib.ptr(y2), _lib.ptr(mean), _lib.ptr(rstd), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_layernorm_fwd2")
    _lib.count(1)
    return y1, y2, mean, rstd


def layernorm_bwd2(dy1, dy2, res, x2d, w1, w2, mean, rstd):
    """``dx = LNbwd(dy1; w1) + LNbwd(dy2; w2) + res`` in one pass, plus the four parameter gradients (fp32)."""
    rows, n = x2d.shape
    dx = torch.empty_like(x2d)
    grads = torch.zeros(4, n, dtype=torch.float32, device=x2d.device)
    rc = _lib.load().sb_layernorm_bwd2(_lib.ptr(dy1), _lib.ptr(dy2), _lib.ptr(res), _lib.ptr(x2d), _lib.ptr(_f32(w1)), _lib.ptr(_f32(w2)),
                                       _lib.ptr(mean), _lib.ptr(rstd), c_int(rows), c_int(n), _lib.ptr(dx), _lib.ptr(grads[0]), _lib.ptr(grads[1]),
                                       _lib.ptr(grads[2]), _lib.ptr(grads[3]), c_int(_lib.sm_count(x2d.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_layernorm_bwd2")
    _lib.count(3)
    return dx, grads[0], grads[1], grads[2], grads[3]


def add3(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(a)
    rc = _lib.load().sb_add3(_lib.ptr(a), _lib.ptr(b), _lib.ptr(c), _lib.ptr(out), c_ll(a.numel()), c_int(_lib.sm_count(a.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_add3")
    _lib.count(1)
    return out


def gelu_fwd(x: torch.Tensor, tanh_form: bool) -> torch.Tensor:
    y = torch.empty_like(x)
    rc = _lib.load().sb_gelu_fwd(_lib.ptr(x), _lib.ptr(y), c_ll(x.numel()), c_int(int(tanh_form)), c_int(_lib.sm_count(x.device)),
                                 _lib.stream_ptr())
    _lib.check_rc(rc, "sb_gelu_fwd")
    _lib.count(1)
    return y


def gelu_bwd(dy: torch.Tensor, x: torch.Tensor, tanh_form: bool) -> torch.Tensor:
    dx = torch.empty_like(x)
    rc = _lib.load().sb_gelu_bwd(_lib.ptr(dy), _lib.ptr(x), _lib.ptr(dx), c_ll(x.numel()), c_int(int(tanh_form)),
                                 c_int(_lib.sm_count(x.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_gelu_bwd")
    _lib.count(1)
    return dx


def gelu_bwd_colsum(dy: torch.Tensor, x: torch.Tensor, tanh_form: bool):
    """``(dx, column sums of dx)`` for contiguous bf16 ``[..., n]`` with ``n % 8 == 0``; the sums are fp32 ``[n]``."""
    n = x.shape[-1]
    rows = x.numel() // n
    dx = torch.empty_like(x)
    sums = torch.zeros(n, dtype=torch.float32, device=x.device)
    rc = _lib.load().sb_gelu_bwd_colsum(_lib.ptr(dy), _lib.ptr(x), _lib.ptr(dx), c_int(rows), c_int(n), c_int(int(tanh_form)), _lib.ptr(sums),
                                        c_int(_lib.sm_count(x.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_gelu_bwd_colsum")
    _lib.count(1)
    return dx, sums


def cross_entropy_fwd(logits: torch.Tensor, target: torch.Tensor):
    """Mean loss over valid rows; returns ``(loss, target_int64, row_lse, inv_valid)`` for :func:`cross_entropy_bwd`."""
    rows, v = logits.shape
    target = target.to(torch.int64)
    inv_valid = 1.0 / (target != -100).sum().clamp_min(1).float()
    row_loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    row_lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
    rc = _lib.load().sb_cross_entropy(_lib.ptr(logits), _lib.ptr(target), c_int(rows), c_int(v), _lib.ptr(inv_valid), _lib.ptr(None),
                                      _lib.ptr(row_loss), _lib.ptr(row_lse), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_cross_entropy")
    _lib.count(1)
    return row_loss.sum() * inv_valid, target, row_lse, inv_valid


def cross_entropy_bwd(logits: torch.Tensor, target: torch.Tensor, row_lse: torch.Tensor, inv_valid: torch.Tensor, dloss: torch.Tensor) -> torch.Tensor:
    """``d loss / d logits`` scaled by the upstream scalar ``dloss`` (a device tensor: no host read)."""
    rows, v = logits.shape
    dlogits = torch.empty_like(logits)
    scale = dloss.detach().float().reshape(1)
    rc = _lib.load().sb_cross_entropy_bwd(_lib.ptr(logits), _lib.ptr(target), c_int(rows), c_int(v), _lib.ptr(row_lse), _lib.ptr(inv_valid),
                                          _lib.ptr(scale), _lib.ptr(dlogits), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_cross_entropy_bwd")
    _lib.count(1)
    return dlogits


def cast_bf16(src: torch.Tensor) -> torch.Tensor:
    """fp32 -> bf16 copy (``numel % 4 == 0``)."""
    dst = torch.empty(src.shape, dtype=torch.bfloat16, device=src.device)
    rc = _lib.load().sb_cast_f32_bf16(_lib.ptr(src), _lib.ptr(dst), c_ll(src.numel()), c_int(_lib.sm_count(src.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_cast_f32_bf16")
    _lib.count(1)
    return dst


def rotary_qk_(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, seq: int, heads: int, head_dim: int, rot: int, sign: float) -> None:
    """In-place rotary embedding of the q and k parts of contiguous bf16 ``qkv`` ``[tokens, heads, 3*head_dim]``."""
    tokens = qkv.numel() // (heads * 3 * head_dim)
    rc = _lib.load().sb_rotary_qk(_lib.ptr(qkv), _lib.ptr(cos), _lib.ptr(sin), c_ll(tokens), c_int(seq), c_int(heads), c_int(head_dim),
                                  c_int(rot), c_float(sign), c_int(_lib.sm_count(qkv.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_rotary_qk")
    _lib.count(1)


def embedding_fwd(table: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """bf16 rows ``table[ids]`` from a bf16 or fp32 table ``[vocab, width]`` (``width % 8 == 0``); ids are checked on the device."""
    vocab, width = table.shape
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    out = torch.empty(flat.numel(), width, dtype=torch.bfloat16, device=table.device)
    bad = torch.zeros(1, dtype=torch.int32, device=table.device)
    rc = _lib.load().sb_embedding_fwd(_lib.ptr(table), c_int(int(table.dtype == torch.bfloat16)), _lib.ptr(flat), c_ll(flat.numel()), c_int(width),
                                      c_int(vocab), _lib.ptr(out), _lib.ptr(bad), c_int(_lib.sm_count(table.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_embedding_fwd")
    _lib.count(1)
    return out.reshape(*ids.shape, width)


def embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, vocab: int, padding_idx: int | None, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 ``[vocab, width]`` gradient of the table: rows of ``dy`` (bf16) summed by id.  ``out`` (contiguous fp32) is cleared and filled."""
    width = dy.shape[-1]
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    d2 = dy.reshape(-1, width).contiguous()
    if out is None:
        out = torch.zeros(vocab, width, dtype=torch.float32, device=dy.device)
    else:
        out.zero_()
    rc = _lib.load().sb_embedding_bwd(_lib.ptr(d2), _lib.ptr(flat), c_ll(flat.numel()), c_int(width), c_int(vocab),
                                      c_ll(-1 if padding_idx is None else padding_idx), _lib.ptr(out), c_int(_lib.sm_count(dy.device)), _lib.stream_ptr())
    _lib.check_rc(rc, "sb_embedding_bwd")
    _lib.count(1)
    return out


DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
ACTIVATION_CODE = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _contiguous_like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of the shape and type of ``t`` (``torch.empty`` with its arguments takes 2 us longer)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _row_stride(t: torch.Tensor):
    """Elements from one row (last dimension) of ``t`` to the next, or ``None`` where the rows do not lie at equal steps."""
    sizes, strides = t.shape, t.stride()
    if sizes[-1] != 1 and strides[-1] != 1:
        return None
    step, expected = None, None
    for size, stride in zip(reversed(sizes[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != expected:
            return None
        expected = stride * size
    return 0 if step is None else step


def _as_rows(*ts: torch.Tensor):
    """``(tensors, rows, n, row strides)``: contiguous tensors as one row, so that a width that is no multiple of a vector costs only the
    last few elements; others as rows where they lie at equal steps, and copied where they do not."""
    if all(t.is_contiguous() for t in ts):
        return ts, 1, ts[0].numel(), (0,) * len(ts)
    steps = [_row_stride(t) for t in ts]
    if None in steps:
        ts = tuple(t if s is not None else t.contiguous() for t, s in zip(ts, steps))
        steps = [_row_stride(t) for t in ts]
    n = ts[0].shape[-1]
    return ts, ts[0].numel() // n, n, steps


def gated_product_fwd(gate: torch.Tensor, up: torch.Tensor, activation: str) -> torch.Tensor:
    """``act(gate) * up`` of two tensors of one shape; the result is contiguous."""
    (gate, up), rows, n, (lg, lu) = _as_rows(gate, up)
    out = _contiguous_like(gate)
    rc = _lib.entry("sb_gated_product_fwd", "pppllll" + "iiip")(
        gate.data_ptr(), up.data_ptr(), out.data_ptr(), lg, lu, rows, n, DTYPE_CODE[gate.dtype], ACTIVATION_CODE[activation], *_lib.place(gate))
    _lib.check_rc(rc, "sb_gated_product_fwd")
    _lib.count(1)
    return out


def gated_product_bwd(dout: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, activation: str, need_gate: bool = True, need_up: bool = True):
    """``(dgate, dup)`` of :func:`gated_product_fwd`, contiguous; ``None`` for one that is not needed."""
    (dout, gate, up), rows, n, (ld, lg, lu) = _as_rows(dout, gate, up)
    dgate = _contiguous_like(gate) if need_gate else None
    dup = _contiguous_like(gate) if need_up else None
    rc = _lib.entry("sb_gated_product_bwd", "ppppplllll" + "iiip")(
        dout.data_ptr(), gate.data_ptr(), up.data_ptr(), None if dgate is None else dgate.data_ptr(), None if dup is None else dup.data_ptr(), ld, lg, lu,
        rows, n, DTYPE_CODE[gate.dtype], ACTIVATION_CODE[activation], *_lib.place(gate))
    _lib.check_rc(rc, "sb_gated_product_bwd")
    _lib.count(1)
    return dgate, dup


def rotary(q, k, inv_freq: torch.Tensor, positions, first: int, interleaved: bool, scale: float, sign: float):
    """Rotated copies of ``q`` ``[B, S, H, D]`` and ``k`` (either may be ``None``), contiguous.

    ``positions`` is an int32 / int64 ``[B, S]`` tensor of any strides, or ``None`` for ``first + s``.
    """
    some = q if q is not None else k
    b, s, _, d = some.shape
    oq = ok = qp = kp = oqp = okp = pp = None
    hq = hk = qb = qs = qh = kb = ks = kh = pb = ps = 0
    if q is not None:
        oq = _contiguous_like(q)
        hq, (qb, qs, qh, _), qp, oqp = q.shape[2], q.stride(), q.data_ptr(), oq.data_ptr()
    if k is not None:
        ok = _contiguous_like(k)
        hk, (kb, ks, kh, _), kp, okp = k.shape[2], k.stride(), k.data_ptr(), ok.data_ptr()
    if positions is not None:
        (pb, ps), pp = positions.stride(), positions.data_ptr()
    rc = _lib.entry("sb_rotary", "pppp" + "llllll" + "ppi" + "llll" + "iiiiiii" + "ff" + "ip")(
        qp, kp, oqp, okp, qb, qs, qh, kb, ks, kh, inv_freq.data_ptr(), pp, positions is not None and positions.dtype == torch.int64, pb, ps, first, b, s, hq, hk,
        d, 2 * inv_freq.numel(), interleaved, DTYPE_CODE[some.dtype], scale, sign, *_lib.place(some))
    _lib.check_rc(rc, "sb_rotary")
    _lib.count(1)
    return oq, ok
