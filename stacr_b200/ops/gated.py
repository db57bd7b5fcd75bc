"""The kernels behind ``nn_ops.gated_linear`` on contiguous bf16 matrices: ``x [M, K]``, weights ``[F, K]``, results ``[M, F]``."""

from __future__ import annotations

import torch

from . import nn_kernels
from .gemm import gemm


def forward(x, wg, wu, bg, bu, activation: str, keep: bool):
    """``(h, gate, up)``; the projections are ``None`` unless ``keep``."""
    g, u = gemm(x, wg, bias=bg, out_dtype=torch.float32), gemm(x, wu, bias=bu, out_dtype=torch.float32)
    h = nn_kernels.gated_product_fwd(g.view(1, -1), u.view(1, -1), activation).view(g.shape).to(torch.bfloat16)
    return (h, g.to(torch.bfloat16), u.to(torch.bfloat16)) if keep else (h, None, None)


def backward_kept(dh, g, u, activation: str):
    """``(dgate, dup)`` from the projections kept by :func:`forward`."""
    dg, du = nn_kernels.gated_product_bwd(dh.view(1, -1), g.view(1, -1), u.view(1, -1), activation)
    return dg.view(g.shape), du.view(g.shape)


def backward_recomputed(dh, x, wg, wu, bg, bu, activation: str):
    """``(dgate, dup)`` with the projections formed again."""
    g, u = gemm(x, wg, bias=bg, out_dtype=torch.float32), gemm(x, wu, bias=bu, out_dtype=torch.float32)
    return tuple(d.to(torch.bfloat16) for d in backward_kept(dh.float(), g, u, activation))


def input_gradient(dg, du, wg, wu):
    """``dgate Wg + dup Wu`` in bf16, summed in fp32."""
    a = gemm(dg, wg, b_mn=True, out_dtype=torch.float32)
    return a.add_(gemm(du, wu, b_mn=True, out_dtype=torch.float32)).to(torch.bfloat16)


def weight_gradients(dg, du, x, gate_dtype, up_dtype, slots, need_gate: bool, need_up: bool):
    """``(dgate^T x, dup^T x)``, fp32 into a slot or for an fp32 weight, bf16 otherwise; ``None`` for one that is not needed."""
    out = []
    for d, dtype, slot, need in ((dg, gate_dtype, slots[0], need_gate), (du, up_dtype, slots[1], need_up)):
        kind = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        out.append(gemm(d, x, a_mn=True, b_mn=True, out=slot, out_dtype=kind) if need else None)
    return out
