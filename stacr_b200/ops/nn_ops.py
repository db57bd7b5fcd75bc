"""Normalisation, activation and loss ops of the model zoo.

For bf16 CUDA tensors these dispatch to the sm_100a kernels in ``csrc/nn_kernels.cu`` (fused
LayerNorm forward/backward with fp32 statistics, GELU forward/backward, fused softmax
cross-entropy that writes the logit gradient in place of a second pass).  Everything else uses
the framework ops, which are also the oracles of the kernel tests.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _lib, gated, nn_kernels


def _kernel_tensor(x: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype == torch.bfloat16


def _differentiable_once(backward):
    """``once_differentiable`` for a backward of kernels: its wrapper is entered only where a graph of the backward is being recorded."""
    recorded = once_differentiable(backward)

    def call(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call


# ------------------------------------------------------------------------------ LayerNorm
class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        from . import nn_kernels

        x2d = x.reshape(-1, x.shape[-1]).contiguous()
        y, mean, rstd = nn_kernels.layernorm_fwd(x2d, weight, bias, eps)
        ctx.save_for_backward(x2d, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        from . import nn_kernels

        x2d, weight, mean, rstd = ctx.saved_tensors
        dy2d = dy.reshape(-1, dy.shape[-1]).contiguous()
        dx, dw, db = nn_kernels.layernorm_bwd(dy2d, x2d, weight, mean, rstd)
        return dx.reshape(dy.shape), dw.to(weight.dtype), (db.to(weight.dtype) if ctx.has_bias else None), None


def layer_norm(x, weight, bias, eps: float = 1e-5):
    if _kernel_tensor(x) and x.shape[-1] % 8 == 0 and x.shape[-1] <= 16384:
        return _LayerNormFn.apply(x, weight, bias, eps)
    return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)


class _ParallelNormsFn(torch.autograd.Function):
    """``(LN1(x), LN2(x), x)`` for a parallel-residual block ``x + f(LN1(x)) + g(LN2(x))``.

    Forward reads ``x`` once for both normalisations.  The third output is ``x`` itself, handed on to the residual sum,
    so that all three gradient streams that meet at ``x`` arrive in this function's backward, which forms
    ``LNbwd(g1) + LNbwd(g2) + g3`` in one kernel instead of two normalisation backwards and two accumulating adds.
    """

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, eps):
        from . import nn_kernels

        x2d = x.reshape(-1, x.shape[-1]).contiguous()
        y1, y2, mean, rstd = nn_kernels.layernorm_fwd2(x2d, w1, b1, w2, b2, eps)
        ctx.save_for_backward(x2d, w1, w2, mean, rstd)
        ctx.x_shape = x.shape
        return y1.reshape(x.shape), y2.reshape(x.shape), x.view_as(x)

    @staticmethod
    def backward(ctx, g1, g2, g3):
        from . import nn_kernels

        x2d, w1, w2, mean, rstd = ctx.saved_tensors

        def flat(g):
            return None if g is None else g.reshape(x2d.shape).to(torch.bfloat16).contiguous()

        g1, g2, g3 = flat(g1), flat(g2), flat(g3)
        if g1 is None:
            g1 = torch.zeros_like(x2d)
        if g2 is None:
            g2 = torch.zeros_like(x2d)
        dx, dw1, db1, dw2, db2 = nn_kernels.layernorm_bwd2(g1, g2, g3, x2d, w1, w2, mean, rstd)
        return dx.reshape(ctx.x_shape), dw1.to(w1.dtype), db1.to(w1.dtype), dw2.to(w2.dtype), db2.to(w2.dtype), None


def parallel_norms_supported(x, w1, b1, w2, b2) -> bool:
    return (_kernel_tensor(x) and x.shape[-1] % 8 == 0 and x.shape[-1] <= 2048 and b1 is not None and b2 is not None
            and w1.shape == w2.shape)


def parallel_layer_norms(x, w1, b1, w2, b2, eps: float = 1e-5):
    """``(LN(x; w1, b1), LN(x; w2, b2), x)``: use the third result as the residual operand (see ``_ParallelNormsFn``)."""
    return _ParallelNormsFn.apply(x, w1, b1, w2, b2, eps)


class _Add3Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, c):
        from . import nn_kernels

        return nn_kernels.add3(a.contiguous(), b.contiguous(), c.contiguous())

    @staticmethod
    def backward(ctx, g):
        return g, g, g


def add3(a, b, c):
    """``a + b + c`` in one pass for bf16 CUDA tensors of one shape."""
    if _kernel_tensor(a) and a.shape == b.shape == c.shape and b.dtype == c.dtype == a.dtype and a.numel() % 8 == 0:
        return _Add3Fn.apply(a, b, c)
    return a + b + c


# ------------------------------------------------------------------------------ column sums handed from producer to consumer
class _ColumnSums:
    """Column sums of a gradient matrix that some kernel produced as a by-product, offered to whoever needs them next.

    The backward of an activation writes ``dX`` and can sum its columns on the way; the backward of the linear layer that
    fed the activation runs next and needs exactly those sums for its bias gradient.  The two are separate autograd nodes,
    so the sums travel through this mailbox keyed by the matrix's storage address, shape and version.  The mailbox keeps
    the matrix itself alive while its entry exists, so the address cannot be recycled for another tensor and a match is
    never a coincidence.  Two slots: ``offered`` holds a producer's by-product and is emptied when it is taken;
    ``remembered`` holds sums that ``bias_grad`` computed itself and stays until the next such computation, so that two
    layers that receive the same gradient tensor (the attention output projection and the MLP output projection of a
    parallel-residual block, whose backward passes are separated by the whole MLP) sum it once.  A lookup that matches
    neither slot leaves the caller to compute the sums.
    """

    def __init__(self):
        self.offered = None        # (key, sums, matrix)
        self.remembered = None

    @staticmethod
    def _key(t: torch.Tensor, cols: int):
        return (t.data_ptr(), t.numel(), cols, t._version, t.device.index)

    def offer(self, matrix: torch.Tensor, sums: torch.Tensor, single_use: bool) -> None:
        entry = (self._key(matrix, sums.numel()), sums, matrix)
        if single_use:
            self.offered = entry
        else:
            self.remembered = entry

    def take(self, matrix: torch.Tensor, cols: int):
        key = self._key(matrix, cols)
        if self.offered is not None and self.offered[0] == key:
            sums, self.offered = self.offered[1], None
            return sums
        if self.remembered is not None and self.remembered[0] == key:
            return self.remembered[1]
        return None

    def clear(self) -> None:
        self.offered = self.remembered = None


column_sums = _ColumnSums()


def bias_grad(g2d: torch.Tensor) -> torch.Tensor:
    """fp32 column sums of a bf16 gradient matrix ``[rows, out]``: taken from the mailbox when its producer left them there."""
    from . import stacr_ops

    hit = column_sums.take(g2d, g2d.shape[1])
    if hit is not None:
        return hit
    sums = stacr_ops.colsum(g2d)
    column_sums.offer(g2d, sums, single_use=False)
    return sums


# ------------------------------------------------------------------------------ GELU
class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tanh_form: bool):
        from . import nn_kernels

        xc = x.contiguous()
        ctx.save_for_backward(xc)
        ctx.tanh_form = tanh_form
        return nn_kernels.gelu_fwd(xc, tanh_form)

    @staticmethod
    def backward(ctx, dy):
        from . import nn_kernels

        (x,) = ctx.saved_tensors
        if x.dim() >= 2 and x.shape[-1] % 8 == 0:
            dx, sums = nn_kernels.gelu_bwd_colsum(dy.contiguous(), x, ctx.tanh_form)
            column_sums.offer(dx, sums, single_use=True)      # the bias gradient of the projection that produced x
            return dx, None
        return nn_kernels.gelu_bwd(dy.contiguous(), x, ctx.tanh_form), None


def gelu(x, approximate: str = "none"):
    if _kernel_tensor(x) and x.numel() % 8 == 0:
        return _GeluFn.apply(x, approximate == "tanh")
    return F.gelu(x, approximate=approximate)


# ------------------------------------------------------------------------------ cross-entropy
class _CrossEntropyFn(torch.autograd.Function):
    """Mean cross-entropy over rows with ``target != -100``.  Forward reads the logits once (loss and row log-sum-exp);
    backward reads them once more and writes the gradient with the upstream scalar folded in."""

    @staticmethod
    def forward(ctx, logits, target):
        from . import nn_kernels

        logits = logits.contiguous()
        loss, tgt, lse, inv_valid = nn_kernels.cross_entropy_fwd(logits, target.contiguous())
        ctx.save_for_backward(logits, tgt, lse, inv_valid)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        from . import nn_kernels

        logits, tgt, lse, inv_valid = ctx.saved_tensors
        return nn_kernels.cross_entropy_bwd(logits, tgt, lse, inv_valid, dloss), None


def cross_entropy(logits, target):
    if _kernel_tensor(logits) and logits.shape[-1] % 8 == 0:
        return _CrossEntropyFn.apply(logits, target)
    return F.cross_entropy(logits.float(), target, ignore_index=-100)


class _PaddedHeadCEFn(torch.autograd.Function):
    """``cross_entropy(hidden @ weight^T, target)`` for a vocabulary that is not a multiple of 8 (GPT-2: 50257).

    Library GEMMs fall back to unaligned legacy kernels when the logits' leading dimension is odd, and the loss kernel needs
    16-byte rows.  Here the logits live in a buffer whose rows are padded to a multiple of 64 columns: the in-tree GEMM writes
    the first ``V`` columns (its output takes a leading dimension), the padding holds a large negative value so that it gets
    no probability, and both backward products read the same padded buffer through strided views.
    """

    @staticmethod
    def forward(ctx, hidden, weight, target):
        from . import nn_kernels
        from .gemm import gemm

        rows, v = hidden.shape[0], weight.shape[0]
        vp = (v + 63) // 64 * 64
        h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
        h = h.contiguous()
        w = weight.detach().to(torch.bfloat16).contiguous()
        logits = torch.empty(rows, vp, dtype=torch.bfloat16, device=hidden.device)
        logits[:, v:].fill_(-30000.0)
        gemm(h, w, out=logits[:, :v])
        loss, tgt, lse, inv_valid = nn_kernels.cross_entropy_fwd(logits, target.contiguous())
        ctx.save_for_backward(h, w, logits, tgt, lse, inv_valid)
        ctx.v, ctx.hidden_dtype, ctx.weight_dtype = v, hidden.dtype, weight.dtype
        return loss

    @staticmethod
    def backward(ctx, dloss):
        from . import nn_kernels
        from .gemm import gemm

        h, w, logits, tgt, lse, inv_valid = ctx.saved_tensors
        d = nn_kernels.cross_entropy_bwd(logits, tgt, lse, inv_valid, dloss)[:, :ctx.v]      # [rows, V] view, rows padded
        dh = gemm(d, w, b_mn=True).to(ctx.hidden_dtype) if ctx.needs_input_grad[0] else None
        dw = gemm(d, h, a_mn=True, b_mn=True, out_dtype=torch.float32).to(ctx.weight_dtype) if ctx.needs_input_grad[1] else None
        return dh, dw, None


def linear_cross_entropy(hidden, weight, target, chunk: int = 0):
    """``cross_entropy(hidden @ weight^T, target)`` evaluated in row chunks to bound the logits workspace."""
    from . import _lib

    padded = hidden.is_cuda and weight.shape[0] % 8 != 0 and hidden.shape[-1] % 8 == 0 and _lib.available() and \
        (hidden.dtype == torch.bfloat16 or torch.is_autocast_enabled())
    if padded:
        def head(h, t):
            return _PaddedHeadCEFn.apply(h, weight, t)
    else:
        def head(h, t):
            return cross_entropy(linear(h, weight), t)
    if not chunk or hidden.shape[0] <= chunk:
        return head(hidden, target)
    valid = (target != -100).sum().clamp_min(1)
    total = hidden.new_zeros((), dtype=torch.float32)
    for lo in range(0, hidden.shape[0], chunk):
        t = target[lo:lo + chunk]
        n = (t != -100).sum()
        total = total + head(hidden[lo:lo + chunk], t).float() * n
    return total / valid


# ------------------------------------------------------------------------------ plain linear layer
class _LinearFn(torch.autograd.Function):
    """``y = x W^T + b`` for a projection that is not compressed.

    All three products run on the in-tree tcgen05 GEMM on bf16 operands (the bf16 copy of the weight is the shadow the
    fused optimizer keeps current, when there is one): forward ``X W^T + b`` with the bias added in the epilogue, the input
    gradient ``dY W`` reading ``W[out, in]`` as an MN-major operand (no transpose is materialised), and the weight gradient
    ``dY^T X`` with fp32 accumulation *and fp32 output*: under autocast a library path produces a bf16 ``dW``, casts it to
    fp32 and, with a flat gradient buffer, copies it into its slot; here the kernel writes fp32 once, straight into the
    slot when a gradient synchroniser has lent one (``weight._sb_grad_out``).
    """

    @staticmethod
    def forward(ctx, x2d, weight, bias):
        # 2-D in, 2-D out: the caller reshapes outside, so that the output is not a view made inside the function
        # (the fused-QKV rotary embedding modifies it in place)
        from ..layers import _bf16_weight

        from .gemm import gemm

        xa = (x2d if x2d.dtype == torch.bfloat16 else x2d.to(torch.bfloat16)).contiguous()
        wb = _bf16_weight(weight).contiguous()
        y = gemm(xa, wb, bias=None if bias is None else bias.detach().float().contiguous())
        ctx.save_for_backward(xa, weight)
        ctx.in_dtype, ctx.bias_dtype = x2d.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        from ..layers import _bf16_weight
        from . import stacr_ops
        from .gemm import gemm

        xa, weight = ctx.saved_tensors
        out_features, in_features = weight.shape
        g = (dy if dy.dtype == torch.bfloat16 else dy.to(torch.bfloat16)).contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = gemm(g, _bf16_weight(weight).contiguous(), b_mn=True).to(ctx.in_dtype)
        if ctx.needs_input_grad[1]:
            slot = getattr(weight, "_sb_grad_out", None) if getattr(weight, "_sb_grad_fresh", False) else None
            if slot is not None and slot.dtype == torch.float32 and weight.dtype == torch.float32:
                weight._sb_grad_fresh = False
            else:
                slot = None
            dw = gemm(g, xa, a_mn=True, b_mn=True, out=slot, out_dtype=torch.float32)
            ready = getattr(weight, "_sb_grad_ready", None) if slot is not None else None
            if ready is not None and not getattr(weight, "_sb_tied", False):
                ready()      # the slot is the gradient: nothing goes back through autograd (it would be cloned)
                dw = None
            elif dw.dtype != weight.dtype:
                dw = dw.to(weight.dtype)
        if ctx.bias_dtype is not None and ctx.needs_input_grad[2]:
            db = bias_grad(g).to(ctx.bias_dtype)
        return dx, dw, db


def linear(x, weight, bias=None):
    """Linear map with the fp32-direct weight gradient on a B200 when the activations are (or autocast makes them) bf16."""
    usable = (x.is_cuda and weight.is_cuda and weight.dim() == 2 and x.shape[-1] % 8 == 0 and weight.shape[0] % 8 == 0 and x.numel() > 0
              and _lib.available()
              and (x.dtype == torch.bfloat16 or (torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16))
              and torch.is_grad_enabled() and weight.requires_grad)
    if usable:
        y = _LinearFn.apply(x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x, weight, bias)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.shape[0])
    return F.linear(x, weight, bias)


# ------------------------------------------------------------------------------ token embedding
class _EmbeddingFn(torch.autograd.Function):
    """bf16 rows of an embedding table; the table's fp32 gradient is scatter-added by an in-tree kernel, straight into the
    slot a gradient synchroniser has lent when there is one.  The rows are read from the optimizer's bf16 copy of the table
    when it exists (what a cast of the fp32 rows would give, without touching the fp32 table)."""

    @staticmethod
    def forward(ctx, weight, ids, padding_idx):
        from ..layers import _bf16_weight
        from . import nn_kernels

        table = _bf16_weight(weight) if getattr(weight, "_bf16_shadow", None) is not None else weight.detach()
        ctx.save_for_backward(ids)
        ctx.weight, ctx.padding_idx = weight, padding_idx
        return nn_kernels.embedding_fwd(table.contiguous(), ids)

    @staticmethod
    def backward(ctx, dy):
        from . import nn_kernels

        (ids,) = ctx.saved_tensors
        weight = ctx.weight
        slot = getattr(weight, "_sb_grad_out", None) if getattr(weight, "_sb_grad_fresh", False) else None
        if slot is not None and slot.dtype == torch.float32 and weight.dtype == torch.float32 and not getattr(weight, "_sb_tied", False):
            weight._sb_grad_fresh = False
        else:
            slot = None
        g = (dy if dy.dtype == torch.bfloat16 else dy.to(torch.bfloat16))
        dw = nn_kernels.embedding_bwd(g, ids, weight.shape[0], ctx.padding_idx, out=slot)
        ready = getattr(weight, "_sb_grad_ready", None) if slot is not None else None
        if ready is not None:
            ready()
            return None, None, None
        return dw.to(weight.dtype), None, None


def embedding(ids, weight, padding_idx=None):
    """Token embedding lookup producing bf16 on a B200 under bf16 autocast (see ``_EmbeddingFn``); the stock op elsewhere."""
    usable = (weight.is_cuda and ids.is_cuda and weight.dim() == 2 and weight.shape[1] % 8 == 0 and _lib.available() and ids.numel() > 0
              and weight.dtype in (torch.float32, torch.bfloat16) and torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16)
    if usable:
        if torch.is_grad_enabled() and weight.requires_grad:
            return _EmbeddingFn.apply(weight, ids, padding_idx)
        from ..layers import _bf16_weight
        from . import nn_kernels

        table = _bf16_weight(weight) if getattr(weight, "_bf16_shadow", None) is not None else weight.detach()
        return nn_kernels.embedding_fwd(table.contiguous(), ids)
    return F.embedding(ids, weight, padding_idx)


# ------------------------------------------------------------------------------ rotary embedding
class _RotaryQKFn(torch.autograd.Function):
    """Rotate q and k inside a fused qkv projection output, in place (the projection does not need its output for backward)."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, seq, heads, head_dim, rot):
        from . import nn_kernels

        nn_kernels.rotary_qk_(qkv, cos, sin, seq, heads, head_dim, rot, 1.0)
        ctx.mark_dirty(qkv)
        ctx.save_for_backward(cos, sin)
        ctx.dims = (seq, heads, head_dim, rot)
        return qkv

    @staticmethod
    def backward(ctx, grad):
        from . import nn_kernels

        cos, sin = ctx.saved_tensors
        g = grad.contiguous()
        if g.data_ptr() == grad.data_ptr():
            g = grad.clone()
        nn_kernels.rotary_qk_(g, cos, sin, *ctx.dims, -1.0)
        return g, None, None, None, None, None, None


def rotary_qk_supported(qkv: torch.Tensor, head_dim: int, rot: int) -> bool:
    return _kernel_tensor(qkv) and qkv.is_contiguous() and rot % 16 == 0 and head_dim % 8 == 0 and rot > 0


def rotary_qk(qkv, cos_half, sin_half, seq: int, heads: int, head_dim: int, rot: int):
    """``qkv``: ``[B, S, heads * 3 * head_dim]`` bf16 (per-head interleaved q|k|v); tables ``[S, rot/2]`` fp32."""
    return _RotaryQKFn.apply(qkv, cos_half, sin_half, seq, heads, head_dim, rot)


# ------------------------------------------------------------------------------ rotary positions of separate q and k
def rotary_frequencies(dim: int, base: float = 10000.0, scaling: dict | None = None, *, seq_len: int | None = None, device=None):
    """``(inv_freq, scale)`` for :func:`rotary`: ``dim / 2`` angular frequencies in 64 bits and the factor on the rotated values.

    ``scaling`` stretches the frequencies to contexts longer than the trained one; its ``rope_type`` (or ``type``) is

    * ``default``: none;
    * ``linear``: every frequency divided by ``factor`` (position interpolation);
    * ``ntk``: the base raised to ``base * factor^(dim / (dim - 2))``, which divides the lowest frequency by ``factor`` and leaves the highest;
    * ``dynamic``: the same with the factor that ``seq_len`` needs, ``factor * seq_len / original - (factor - 1)``, beyond the original length;
    * ``yarn``: divided by ``factor`` where fewer than ``beta_slow`` turns fit into the original length, kept where more than ``beta_fast``
      do, linear in between; ``scale = 0.1 ln(factor) + 1`` unless ``attention_factor`` is given;
    * ``llama3``: divided where the wavelength exceeds ``original / low_freq_factor``, kept below ``original / high_freq_factor``, and
      blended in between.

    ``original`` is ``original_max_position_embeddings``.
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary dimension must be positive and even, got {dim}")
    if base <= 0:
        raise ValueError(f"rotary base must be positive, got {base}")
    index = torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim
    inv = float(base) ** -index
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind in (None, "default"):
        return inv, 1.0
    if kind not in ("linear", "ntk", "dynamic", "yarn", "llama3"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    if "factor" not in scaling:
        raise ValueError(f"rotary scaling {kind!r} needs a factor")
    factor = float(scaling["factor"])
    if factor < 1:
        raise ValueError(f"rotary scaling factor must be at least 1, got {factor}")
    original = scaling.get("original_max_position_embeddings")
    if kind in ("dynamic", "yarn", "llama3") and not original:
        raise ValueError(f"rotary scaling {kind!r} needs original_max_position_embeddings")
    if kind == "linear":
        return inv / factor, 1.0
    if kind in ("ntk", "dynamic"):
        if kind == "dynamic":
            factor = factor * seq_len / original - (factor - 1) if seq_len is not None and seq_len > original else 1.0
        stretched = float(base) * factor ** (dim / (dim - 2)) if dim > 2 else float(base)
        return stretched ** -index, 1.0
    if kind == "yarn":
        if base <= 1:
            raise ValueError(f"rotary scaling 'yarn' needs a base above 1, got {base}")

        def pair_with(turns):       # the (real) pair index whose frequency makes this many turns over the original length
            return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_with(float(scaling.get("beta_fast", 32)))), 0)
        high = min(math.ceil(pair_with(float(scaling.get("beta_slow", 1)))), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64, device=device) - low) / max(high - low, 1e-3)).clamp(0, 1)
        attention = scaling.get("attention_factor")
        return inv / factor * ramp + inv * (1 - ramp), float(attention) if attention is not None else 0.1 * math.log(factor) + 1.0
    low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
    if high <= low:
        raise ValueError(f"high_freq_factor must exceed low_freq_factor, got {high} and {low}")
    blend = ((original * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)      # wavelengths in the original length
    return inv / factor * (1 - blend) + inv * blend, 1.0


def _rotary_reference(x, angle, interleaved: bool, scale: float):
    """The framework-op form of :func:`rotary` for one tensor: ``angle`` is ``[B or 1, S, rot / 2]`` in 64 bits."""
    wide = x.dtype if x.dtype in (torch.float32, torch.float64) else torch.float32
    cos, sin = (scale * angle.cos()).to(wide)[:, :, None], (scale * angle.sin()).to(wide)[:, :, None]
    rot = 2 * angle.shape[-1]
    r, rest = x[..., :rot].to(wide), x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, dim=-1)
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, dim=-1).flatten(-2) if interleaved else torch.cat(y, dim=-1)
    return torch.cat((y.to(x.dtype), rest), dim=-1)


class _RotaryFn(torch.autograd.Function):
    """The rotation of q and k; its gradient is the rotation by the opposite angle of the outputs' gradients."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, first, interleaved, scale):
        ctx.save_for_backward(inv_freq, positions)
        ctx.set_materialize_grads(False)
        ctx.first, ctx.interleaved, ctx.scale = first, interleaved, scale
        with _lib.on_device(q):
            out = nn_kernels.rotary(_heads(q), _heads(k), inv_freq, positions, first, interleaved, scale, 1.0)
        frozen = [t for t, needed in zip(out, ctx.needs_input_grad) if t is not None and not needed]
        if frozen:
            ctx.mark_non_differentiable(*frozen)
        return out

    @staticmethod
    @_differentiable_once
    def backward(ctx, gq, gk):
        inv_freq, positions = ctx.saved_tensors
        gq = _heads(gq) if ctx.needs_input_grad[0] else None
        gk = _heads(gk) if ctx.needs_input_grad[1] else None
        if gq is not None or gk is not None:
            with _lib.on_device(inv_freq):
                gq, gk = nn_kernels.rotary(gq, gk, inv_freq, positions, ctx.first, ctx.interleaved, ctx.scale, -1.0)
        return gq, gk, None, None, None, None, None


def _heads(t):
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def rotary(q, k, inv_freq, positions=None, *, interleaved: bool = False, scale: float = 1.0):
    """Rotary positions: ``(q', k')`` for ``q`` ``[B, S, heads, D]`` and ``k`` ``[B, S, kv_heads, D]`` (or ``None``).

    ``inv_freq`` (see :func:`rotary_frequencies`) has ``rot / 2`` angular frequencies; the first ``rot <= D`` values of a head are
    turned, as pairs ``(i, i + rot / 2)`` or, interleaved, ``(2 i, 2 i + 1)``, and the rest is copied.  Pair ``i`` at position ``p`` is
    turned by ``p * inv_freq[i]`` and multiplied by ``scale``; the angle is formed in 64 bits, and ``inv_freq`` receives no gradient.
    ``positions`` is ``None`` (``0 .. S-1``), an int (the first token's position), or an integer tensor ``[S]``, ``[1, S]``, ``[B, 1]``
    or ``[B, S]``.  Inputs may have any strides (a transposed ``[B, heads, S, D]`` view is read in place); results are contiguous.
    """
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("rotary expects q and k as [batch, sequence, heads, head_dim]")
    b, s, _, d = q.shape
    dtype = q.dtype
    if k is not None:
        kb, ks, _, kd = k.shape
        if kb != b or ks != s or kd != d:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, sequence or head_dim")
        if k.dtype is not dtype or k.device != q.device:
            raise ValueError("q and k must have one dtype and one device")
    if not dtype.is_floating_point:
        raise TypeError(f"rotary expects floating-point heads, got {dtype}")
    if inv_freq.dim() != 1 or not inv_freq.dtype.is_floating_point or not 0 < 2 * inv_freq.numel() <= d:
        raise ValueError(f"inv_freq must hold 1 to {d // 2} frequencies, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    first = 0
    if isinstance(positions, int):
        first, positions = positions, None
    elif positions is not None:
        kind, shape = positions.dtype, tuple(positions.shape)
        if kind.is_floating_point or kind.is_complex or kind is torch.bool:
            raise TypeError(f"positions must be integers, got {kind}")
        if shape != (b, s):
            if len(shape) not in (1, 2) or shape[-1] not in (1, s) or (len(shape) == 2 and shape[0] not in (1, b)):
                raise ValueError(f"positions {shape} do not fit [{b}, {s}]")
            positions = positions.expand(b, s)
        if positions.device != q.device:
            positions = positions.to(q.device)
    inv = inv_freq
    if inv.dtype is not torch.float64 or inv.device != q.device or inv.requires_grad or not inv.is_contiguous():
        inv = inv.detach().to(device=q.device, dtype=torch.float64).contiguous()
    if q.is_cuda and dtype in nn_kernels.DTYPE_CODE and d <= 512 and (q.numel() or (k is not None and k.numel())):
        if positions is not None and positions.dtype not in (torch.int32, torch.int64):
            positions = positions.to(torch.int64)
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            return _RotaryFn.apply(q, k, inv, positions, first, bool(interleaved), float(scale))
        with _lib.on_device(q):
            return nn_kernels.rotary(_heads(q), _heads(k), inv, positions, first, bool(interleaved), float(scale), 1.0)
    where = torch.arange(first, first + s, device=q.device)[None] if positions is None else positions
    angle = where.to(torch.float64)[..., None] * inv
    return _rotary_reference(q, angle, interleaved, scale), None if k is None else _rotary_reference(k, angle, interleaved, scale)


# ------------------------------------------------------------------------------ gated activation
_ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda x: F.gelu(x, approximate="tanh")}


def _check_activation(activation: str) -> None:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; choose from {sorted(_ACTIVATIONS)}")


class _GatedProductFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, activation):
        ctx.save_for_backward(gate, up)
        ctx.activation = activation
        with _lib.on_device(gate):
            return nn_kernels.gated_product_fwd(gate, up, activation)

    @staticmethod
    @_differentiable_once
    def backward(ctx, dout):
        gate, up = ctx.saved_tensors
        need_gate, need_up, _ = ctx.needs_input_grad
        with _lib.on_device(gate):
            dgate, dup = nn_kernels.gated_product_bwd(dout, gate, up, ctx.activation, need_gate, need_up)
        return dgate, dup, None


def gated_product(gate, up, activation: str = "silu"):
    """``act(gate) * up`` for two tensors of one shape, in fp32 and rounded once; ``activation``: ``silu``, ``gelu`` or ``gelu_tanh``.

    bf16, fp16 and fp32 CUDA tensors take one kernel forward and one backward; rows may be strided (the halves of one fused
    projection).  Elsewhere, and for mixed types, the framework ops.
    """
    _check_activation(activation)
    if gate.shape != up.shape:
        raise ValueError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} differ in shape")
    if gate.is_cuda and gate.dtype is up.dtype and gate.dtype in nn_kernels.DTYPE_CODE and gate.device == up.device and gate.numel() and gate.dim():
        if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
            return _GatedProductFn.apply(gate, up, activation)
        with _lib.on_device(gate):
            return nn_kernels.gated_product_fwd(gate, up, activation)
    return _ACTIVATIONS[activation](gate) * up


# ------------------------------------------------------------------------------ gated feed-forward: both projections and the product
def _take_slot(weight):
    """The fp32 buffer a gradient synchroniser has lent for this weight's gradient, or ``None``."""
    slot = getattr(weight, "_sb_grad_out", None) if getattr(weight, "_sb_grad_fresh", False) else None
    if slot is None or slot.dtype != torch.float32 or weight.dtype != torch.float32 or not slot.is_contiguous() or slot.data_ptr() % 16:
        return None         # the gradient then goes back through autograd, and the synchroniser moves it
    weight._sb_grad_fresh = False
    return slot


def _hand_over(weight, dw, slot):
    """What goes back through autograd for a weight whose gradient ``dw`` was written, into ``slot`` if there is one."""
    ready = getattr(weight, "_sb_grad_ready", None) if slot is not None else None
    if ready is not None and not getattr(weight, "_sb_tied", False):
        ready()
        return None
    return dw if dw.dtype == weight.dtype else dw.to(weight.dtype)


def _operand(t):
    """``t`` as the tensor-core kernels read it: bf16, contiguous and on a 16-byte boundary (a copy where it is not)."""
    t = (t if t.dtype == torch.bfloat16 else t.detach().to(torch.bfloat16)).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _bf16_operand(weight):
    if weight.dtype == torch.bfloat16:
        return _operand(weight)
    from ..layers import _bf16_weight

    return _operand(_bf16_weight(weight))


def _weight_gradient_buffer(weight, slot):
    """Where a weight's gradient is formed: the lent slot, else a new matrix, fp32 unless the weight itself is bf16."""
    if slot is not None:
        return slot
    if weight.dtype in (torch.bfloat16, torch.float32) and weight.is_contiguous():
        return torch.empty_like(weight)
    return weight.new_empty(weight.shape, dtype=torch.bfloat16 if weight.dtype == torch.bfloat16 else torch.float32)


class _GatedLinearFn(torch.autograd.Function):
    """``h = act(x Wg^T + bg) * (x Wu^T + bu)`` on bf16 operands.

    Kept for backward: ``x``, and the two factors ``A = up act'(gate)``, ``B = act(gate)`` of ``dgate = dh A``, ``dup = dh B`` in 24 bits
    each, six bytes a feature, which is what separate layers keep (gate, act(gate) and up in bf16).  With ``recompute`` only ``x``.
    """

    @staticmethod
    def forward(ctx, x2d, gate_weight, up_weight, gate_bias, up_bias, activation, recompute):
        with _lib.on_device(x2d):
            xa = _operand(x2d)
            h, kept = gated.forward(xa, _bf16_operand(gate_weight), _bf16_operand(up_weight), _f32_bias(gate_bias), _f32_bias(up_bias), activation,
                                    keep=not recompute)
        ctx.save_for_backward(xa, gate_weight, up_weight, gate_bias, up_bias, kept)
        ctx.activation, ctx.in_dtype = activation, x2d.dtype
        return h

    @staticmethod
    @_differentiable_once
    def backward(ctx, dh):
        xa, gate_weight, up_weight, gate_bias, up_bias, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dbg = dbu = None
        with _lib.on_device(xa):
            dh = _operand(dh)
            same = gate_weight is up_weight       # one weight in both places receives two gradients: neither may use its slot
            gslot = _take_slot(gate_weight) if need[1] and not same else None
            uslot = _take_slot(up_weight) if need[2] and not same else None
            dwg = _weight_gradient_buffer(gate_weight, gslot) if need[1] else None
            dwu = _weight_gradient_buffer(up_weight, uslot) if need[2] else None
            d, dx = gated.backward(dh, xa, _bf16_operand(gate_weight), _bf16_operand(up_weight), _f32_bias(gate_bias), _f32_bias(up_bias), ctx.activation,
                                   kept, need[0], dwg, dwu)
            if dx is not None and dx.dtype != ctx.in_dtype:
                dx = dx.to(ctx.in_dtype)
            if dwg is not None:
                dwg = _hand_over(gate_weight, dwg, gslot)
            if dwu is not None:
                dwu = _hand_over(up_weight, dwu, uslot)
            if gate_bias is not None and need[3]:
                from . import stacr_ops

                dbg = stacr_ops.colsum(d[0]).to(gate_bias.dtype)
            if up_bias is not None and need[4]:
                from . import stacr_ops

                dbu = stacr_ops.colsum(d[1]).to(up_bias.dtype)
        return dx, dwg, dwu, dbg, dbu, None, None


def _f32_bias(bias):
    return None if bias is None else bias.detach().float().contiguous()


def gated_linear_supported(x, gate_weight, up_weight) -> bool:
    """Whether :func:`gated_linear` takes its kernels for these operands (bf16 activations, or bf16 autocast, on one GPU)."""
    if not x.is_cuda or gate_weight.dim() != 2:
        return False
    f, k = gate_weight.shape
    return (f % 8 == 0 and k % 8 == 0 and f > 0 and x.numel() > 0 and x.device == gate_weight.device == up_weight.device
            and (x.dtype is torch.bfloat16 or (torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16)))


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, *, activation: str = "silu", recompute: bool = False):
    """``act(x Wg^T + bg) * (x Wu^T + bu)``: the first half of a gated feed-forward block, ``[..., K]`` to ``[..., F]``.

    Weights are ``[F, K]``; ``activation``: ``silu``, ``gelu`` or ``gelu_tanh``.  bf16 activations (or bf16 autocast) on a GPU with
    ``K`` and ``F`` multiples of 8 run on tensor cores, projections, activation and product in one kernel; elsewhere the framework ops.
    Backward keeps two factors of six bytes a feature together, or with ``recompute`` only ``x`` and forms the projections again.
    """
    _check_activation(activation)
    if gate_weight.dim() != 2 or gate_weight.shape != up_weight.shape or x.dim() < 1 or x.shape[-1] != gate_weight.shape[1]:
        raise ValueError(f"weights {tuple(gate_weight.shape)} and {tuple(up_weight.shape)} do not project x {tuple(x.shape)}")
    for bias in (gate_bias, up_bias):
        if bias is not None and tuple(bias.shape) != (gate_weight.shape[0],):
            raise ValueError(f"bias {tuple(bias.shape)} does not fit {gate_weight.shape[0]} outputs")
    if not gated_linear_supported(x, gate_weight, up_weight):
        return gated_product(linear(x, gate_weight, gate_bias), linear(x, up_weight, up_bias), activation)
    x2d = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and (x.requires_grad or gate_weight.requires_grad or up_weight.requires_grad
                                    or any(b is not None and b.requires_grad for b in (gate_bias, up_bias))):
        h = _GatedLinearFn.apply(x2d, gate_weight, up_weight, gate_bias, up_bias, activation, bool(recompute))
    else:
        with _lib.on_device(x):
            h = gated.forward(_operand(x2d), _bf16_operand(gate_weight), _bf16_operand(up_weight), _f32_bias(gate_bias), _f32_bias(up_bias), activation,
                              keep=False)[0]
    return h if x.dim() == 2 else h.reshape(*x.shape[:-1], gate_weight.shape[0])
