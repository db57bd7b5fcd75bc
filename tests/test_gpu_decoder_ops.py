"""Rotary positions, gated feed-forward and gradient clipping kernels against their definitions in 64 bits.

Tolerances count roundings: a result rounded to a type is off by at most half a step of it (``HALF``, relative), and every
rounded intermediate carries its half step through the formula (see ``gated_bounds``).
"""

import pytest
import torch
from torch.nn import functional as F

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}   # half a step among the subnormals, or what is flushed
ACTS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}


def inside(got, want, bound, what=""):
    if not want.numel():
        return
    excess = (got.double() - want).abs() - bound
    worst = float(excess.max())
    assert worst <= 0, f"{what}: off by {worst:.3g} more than its bound at {int(excess.argmax())}"


# ------------------------------------------------------------------------------------------------ rotary
def turned(x, positions, inv, interleaved, scale=1.0):
    x, rot = x.double(), 2 * inv.numel()
    theta = positions.double()[..., None] * inv
    head = x[..., :rot].unflatten(-1, (-1, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * torch.polar(torch.full_like(theta, scale), theta)[:, :, None])
    return torch.cat(((z if interleaved else z.transpose(-1, -2)).flatten(-2), x[..., rot:]), -1)


def rotary_bound(x, positions, inv, interleaved, scale):
    """Half a step of the result, plus fp32 work: the turn's fraction (2^-25 of half a turn: pi 2^-25 radians), sine and cosine (2 steps
    of 2^-24 each), their scaling, two products and a sum: below 10 2^-24 (|x1| + |x2|) scale."""
    rot = 2 * inv.numel()
    head = x.double()[..., :rot].abs()
    pairs = head.unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(*head.shape[:-1], rot // 2, 2).flatten(-2) if interleaved \
        else head.unflatten(-1, (2, -1)).sum(-2, keepdim=True).expand(*head.shape[:-1], 2, rot // 2).flatten(-2)
    bound = turned(x, positions, inv, interleaved, scale).abs() * HALF[x.dtype] + TINY[x.dtype]
    bound[..., :rot] += 10 * 2.0 ** -24 * scale * pairs
    bound[..., rot:] = 0
    return bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,hq,hk,d,rot", [(1, 1, 1, 1, 2, 2), (3, 7, 4, 2, 64, 64), (2, 65, 28, 4, 128, 128), (1, 130, 5, 5, 80, 20), (2, 9, 3, 1, 30, 6),
                                             (64, 1, 32, 8, 64, 64), (1, 2049, 2, 1, 96, 48),
                                             (2, 5, 1, 1, 512, 510), (1, 3, 2, 1, 509, 506), (1, 2, 1, 1, 520, 520), (1, 3000, 71, 1, 16, 8)])
def test_rotary_forward_and_backward(b, s, hq, hk, d, rot, interleaved, dtype):
    from stacr_b200.ops import nn_ops

    torch.manual_seed(s + d)
    inv, _ = nn_ops.rotary_frequencies(rot, 500000.0, device="cuda")
    q = torch.randn(b, s, hq, d, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(b, s, hk, d, device="cuda").to(dtype).requires_grad_()
    pos = torch.randint(0, 2 ** 20, (b, s), device="cuda")
    out = nn_ops.rotary(q, k, inv, pos, interleaved=interleaved, scale=1.25)
    grads = [torch.randn_like(t) for t in out]
    back = torch.autograd.grad(out, (q, k), grads)
    for x, y, g, dx in zip((q, k), out, grads, back):
        x = x.detach()
        inside(y.detach(), turned(x, pos, inv, interleaved, 1.25), rotary_bound(x, pos, inv, interleaved, 1.25), "forward")
        inside(dx, turned(g, -pos, inv, interleaved, 1.25), rotary_bound(g, -pos, inv, interleaved, 1.25), "backward")


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_reads_views_of_any_stride(interleaved):
    from stacr_b200.ops import nn_ops

    inv, _ = nn_ops.rotary_frequencies(32, device="cuda")
    fused = torch.randn(2, 11, 6, 3 * 64 + 1, device="cuda").bfloat16()
    views = {"split of a projection": fused[..., 64:128], "odd offset": fused[..., 1:65], "transposed": torch.randn(2, 6, 11, 64, device="cuda").bfloat16().transpose(1, 2),
             "every other value": torch.randn(2, 11, 6, 128, device="cuda").bfloat16()[..., ::2], "broadcast": torch.randn(2, 11, 1, 64, device="cuda").bfloat16().expand(2, 11, 6, 64),
             "reversed batch": fused.flip(0)[..., :64]}
    for name, q in views.items():
        for k in (None, fused[..., :64]):
            got = nn_ops.rotary(q, k, inv, 17, interleaved=interleaved)
            want = nn_ops.rotary(q.contiguous(), None if k is None else k.contiguous(), inv, 17, interleaved=interleaved)
            assert torch.equal(got[0], want[0]) and (k is None or torch.equal(got[1], want[1])), name
            assert got[0].is_contiguous()


def test_rotary_positions_types_offsets_and_partial_gradients():
    from stacr_b200.ops import nn_ops

    inv, _ = nn_ops.rotary_frequencies(64, device="cuda")
    q = torch.randn(3, 5, 2, 64, device="cuda", requires_grad=True)
    k = torch.randn(3, 5, 1, 64, device="cuda", requires_grad=True)
    base = nn_ops.rotary(q, k, inv, 4)
    for pos in (torch.arange(4, 9, device="cuda"), torch.arange(4, 9, device="cuda", dtype=torch.int32)[None], torch.arange(4, 9, device="cuda").expand(3, 5),
                torch.arange(4, 9), torch.arange(4, 9, dtype=torch.int16, device="cuda"), torch.arange(8, 18, 2, device="cuda").mul(0).add(torch.arange(4, 9, device="cuda"))):
        again = nn_ops.rotary(q, k, inv, pos)
        assert torch.equal(again[0], base[0]) and torch.equal(again[1], base[1])
    for at in (-3, 2 ** 31 + 5, 2 ** 40):
        got = nn_ops.rotary(q, None, inv, at)[0].detach()
        where = torch.arange(at, at + 5, device="cuda")[None]
        if abs(at) < 2 ** 32:
            inside(got, turned(q.detach(), where, inv, False), rotary_bound(q.detach(), where, inv, False, 1.0))
        assert torch.equal(got, nn_ops.rotary(q, None, inv, where)[0])
    # a gradient for one of the two only, and for a frozen one none
    (dk,) = torch.autograd.grad(nn_ops.rotary(q, k, inv)[1].sum(), k)
    (dq,) = torch.autograd.grad(nn_ops.rotary(q, k.detach(), inv)[0].sum(), q)
    assert torch.isfinite(dk).all() and torch.isfinite(dq).all()
    out = nn_ops.rotary(q.detach(), k, inv)
    assert not out[0].requires_grad and out[1].requires_grad
    with pytest.raises(RuntimeError):
        (g,) = torch.autograd.grad(nn_ops.rotary(q, None, inv)[0].sum(), q, create_graph=True)
        g.sum().backward()


def test_gated_operators_refuse_second_derivatives():
    from stacr_b200.ops import nn_ops

    x, wg, wu, _, _, _ = gated_inputs(9, 16, 24)
    for call in (lambda t: nn_ops.gated_product(t, t), lambda t: nn_ops.gated_linear(t, wg, wu)):
        leaf = x.detach().clone().requires_grad_()
        (g,) = torch.autograd.grad(call(leaf).float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().sum().backward()


def test_rotary_offsets_beyond_32_bits():
    from stacr_b200.ops import nn_ops

    inv, _ = nn_ops.rotary_frequencies(64, device="cuda")
    cache = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    q = cache.as_strided((2, 3, 2, 64), (2 ** 31, 128, 64, 1))
    q.copy_(torch.randn(2, 3, 2, 64, device="cuda"))
    assert torch.equal(nn_ops.rotary(q, None, inv)[0], nn_ops.rotary(q.clone(memory_format=torch.contiguous_format), None, inv)[0])


def test_rotary_gradient_against_differences():
    from stacr_b200.ops import nn_ops

    torch.manual_seed(3)
    inv, _ = nn_ops.rotary_frequencies(8, device="cuda")
    q = torch.randn(1, 3, 2, 8, device="cuda", requires_grad=True)
    w = torch.randn(1, 3, 2, 8, device="cuda")
    (dq,) = torch.autograd.grad((nn_ops.rotary(q, None, inv, 9)[0] * w).sum(), q)
    for i in (0, 5, 17, 40):
        e = torch.zeros_like(q).view(-1)
        e[i] = 0.5
        e = e.view_as(q)
        up, down = (((nn_ops.rotary(q.detach() + s * e, None, inv, 9)[0].double() * w).sum()) for s in (1, -1))
        # the map is linear: the quotient is exact up to fp32 roundings of 48 values of size 4
        assert abs(float(up - down) - float(dq.view(-1)[i])) < 48 * 4 * 2.0 ** -22


# ------------------------------------------------------------------------------------------------ gated activation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("shape,split", [((1, 1), False), ((7, 33), True), ((5, 3, 1003), True), ((64, 4096), False), ((300, 688), True), ((3, 100001), False)])
def test_gated_product_forward_and_backward(shape, split, act, dtype):
    from stacr_b200.ops import nn_ops

    torch.manual_seed(shape[-1])
    n = shape[-1]
    both = (torch.randn(*shape[:-1], 2 * n, device="cuda") * 3).to(dtype)
    gate, up = both[..., :n], both[..., n:]
    if not split:
        gate, up = gate.contiguous(), up.contiguous()
    gate, up = gate.detach().requires_grad_(), up.detach().requires_grad_()
    out = nn_ops.gated_product(gate, up, act)
    dout = torch.randn(shape, device="cuda").to(dtype)
    dgate, dup = torch.autograd.grad(out, (gate, up), dout)
    g, u = gate.detach().double().requires_grad_(), up.detach().double().requires_grad_()
    want = ACTS[act](g) * u
    wg, wu = torch.autograd.grad(want, (g, u), dout.double())
    # activation and derivative in fp32: at most 16 roundings of values bounded by max(1.13, |g|)
    size, d = g.detach().abs().clamp_min(1.2), dout.double().abs()
    fp = 16 * 2.0 ** -24
    inside(out.detach(), want.detach(), want.detach().abs() * HALF[dtype] + fp * size * u.detach().abs() + TINY[dtype], "out")
    inside(dup, wu, wu.abs() * HALF[dtype] + fp * size * d + TINY[dtype], "dup")
    inside(dgate, wg, wg.abs() * HALF[dtype] + fp * size * (u.detach() * d).abs() + TINY[dtype], "dgate")


@pytest.mark.parametrize("act", list(ACTS))
def test_gated_product_extreme_values(act):
    from stacr_b200.ops import nn_ops

    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 87.0, -87.0, 89.0, -89.0, 1e4, -1e4, 3e38, float("inf"), float("nan")], device="cuda")
    one = torch.ones_like(g)
    got, want = nn_ops.gated_product(g, one, act), ACTS[act](g.double())
    finite = torch.isfinite(want)
    # The sigmoid (distribution function) s of a far negative x is flushed to zero below 2^-126, or where e^-x passes fp32's largest
    # value (s < 2^-127): x s is then off by at most |x| 2^-126.
    inside(got[finite], want[finite], want[finite].abs() * 2.0 ** -19 + g[finite].double().abs().clamp_min(1) * 2.0 ** -126)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf() | (want.abs() > 3.5e38))


def test_gated_product_partial_gradients_strides_and_mixed_types():
    from stacr_b200.ops import nn_ops

    gate = torch.randn(6, 40, device="cuda").bfloat16()
    up = torch.randn(40, 6, device="cuda").bfloat16().t().requires_grad_()
    out = nn_ops.gated_product(gate, up)
    (dup,) = torch.autograd.grad(out, up, torch.ones(1, 1, device="cuda").bfloat16().expand(6, 40))
    inside(dup, F.silu(gate.double()), F.silu(gate.double()).abs() * HALF[torch.bfloat16] + 1e-6)
    mixed = nn_ops.gated_product(gate, up.detach().float())
    assert mixed.dtype == torch.float32 and mixed.shape == (6, 40)
    assert nn_ops.gated_product(gate[:0], up.detach()[:0]).shape == (0, 40)


# ------------------------------------------------------------------------------------------------ gated linear
def gated_exact(x, wg, wu, bg, bu, dh, act):
    leaves = [t.detach().double().requires_grad_() for t in (x, wg, wu, bg, bu)]
    xd, g_w, u_w, g_b, u_b = leaves
    g, u = F.linear(xd, g_w, g_b), F.linear(xd, u_w, u_b)
    h = ACTS[act](g) * u
    grads = torch.autograd.grad(h, leaves, dh.double())
    return g.detach(), u.detach(), h.detach(), grads


def gated_bounds(x, wg, wu, bg, bu, dh, act, g, u, keep):
    """Bounds of (h, dx, dWg, dWu, dbg, dbu), element by element.

    A projection is off by its fp32 summation, at most (K + 2) 2^-24 times the sum of its terms' sizes; |act'| <= 1.13, |act''| <= 1.
    The factors that are kept for backward are cut to 24 bits (one step: 2^-15).  The derivative's products are rounded to bf16 before they are
    multiplied again; sums over F or the tokens in fp32 add their length times 2^-24; every result is rounded once.
    """
    e, f32 = HALF[torch.bfloat16], 2.0 ** -24
    X, WG, WU, D = (t.detach().double().abs() for t in (x, wg, wu, dh))
    k, n = X.shape[1], X.shape[0]
    acc = (k + 2) * f32
    eg = acc * (X @ WG.t() + bg.detach().double().abs())
    eu = acc * (X @ WU.t() + bu.detach().double().abs())
    gd = g.clone().requires_grad_()
    a = ACTS[act](gd)
    (da,) = torch.autograd.grad(a.sum(), gd)
    a, da, U = a.detach().abs(), da.abs(), u.abs()
    fp = 16 * f32 * g.abs().clamp_min(1.2)
    bh = (a * U) * e + (1.13 * eg + fp) * (U + eu) + a * eu + 1e-30
    ea, eda = 1.13 * eg + fp, eg + fp
    kept = 2.0 ** -15 if keep else 0.0
    edg = D * ((eda * (U + eu)) + da * eu + kept * (U + eu) * (da + eda))
    edu = D * (ea + kept * (a + ea))
    DG, DU = D * U * da, D * a
    edg, edu = edg + e * (DG + edg) + 1e-35, edu + e * (DU + edu) + 1e-35
    f = WG.shape[0]
    raw = (DG + edg) @ WG + (DU + edu) @ WU
    bdx = edg @ WG + edu @ WU + (2 * f + 2) * f32 * raw + e * raw
    out = [bh, bdx]
    for ED, S in ((edg, DG), (edu, DU)):
        raw = (S + ED).t() @ X
        out.append(ED.t() @ X + (n + 2) * f32 * raw + e * raw)
    for ED, S in ((edg, DG), (edu, DU)):
        raw = (S + ED).sum(0)
        out.append(ED.sum(0) + (n + 2) * f32 * raw + e * raw)
    return out


def gated_inputs(m, k, f, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    return [normal(m, k), normal(f, k, std=0.05), normal(f, k, std=0.05), normal(f, std=0.5), normal(f, std=0.5), normal(m, f, std=0.1)]


GATED_SHAPES = [(1, 8, 8), (1, 2048, 688), (2, 64, 136), (7, 1000, 264), (17, 512, 1000), (33, 1536, 896), (64, 72, 128), (65, 200, 2056), (127, 256, 688),
                (129, 512, 520), (254, 256, 688), (257, 1032, 384), (1000, 264, 1096), (1531, 768, 2048), (4100, 264, 520), (5000, 72, 136),
                # each token count of the kernel for some tokens, with whole and ragged features
                (16, 1024, 16384), (13, 1032, 16392), (32, 256, 14336), (27, 264, 14344), (64, 256, 14336), (50, 264, 14344), (128, 64, 256)]


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("m,k,f", GATED_SHAPES)
def test_gated_linear_forward_and_backward(m, k, f, recompute):
    from stacr_b200.ops import nn_ops

    act = list(ACTS)[(m + k + f) // 8 % 3]
    x, wg, wu, bg, bu, dh = gated_inputs(m, k, f, seed=m + k + f)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = nn_ops.gated_linear(*leaves, activation=act, recompute=recompute)
    assert h.dtype == torch.bfloat16 and h.shape == (m, f)
    got = torch.autograd.grad(h, leaves, dh)
    g, u, want, grads = gated_exact(*leaves, dh, act)
    bounds = gated_bounds(*leaves, dh, act, g, u, keep=not recompute)
    for name, a, b, bound in zip(("h", "dx", "dWg", "dWu", "dbg", "dbu"), (h.detach(), *got), (want, *grads), bounds):
        inside(a, b, bound, name)
    with torch.no_grad():
        assert torch.equal(nn_ops.gated_linear(*leaves, activation=act), h)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16, 24, 31, 32, 40, 63, 64, 66, 100, 128])
def test_gated_linear_without_gradient_at_token_counts(m):
    from stacr_b200.ops import nn_ops

    x, wg, wu, bg, bu, dh = gated_inputs(m, 520, 776, seed=m)
    g, u, want, _ = gated_exact(x, wg, wu, bg, bu, dh, "silu")
    bound = gated_bounds(x, wg, wu, bg, bu, dh, "silu", g, u, keep=False)[0]
    inside(nn_ops.gated_linear(x, wg, wu, bg, bu), want, bound)
    # without biases, and rows of an embedding's view as x
    wide = torch.randn(m, 2 * 520, device="cuda").bfloat16()
    a, b = nn_ops.gated_linear(wide[:, 520:], wg, wu), nn_ops.gated_linear(wide[:, 520:].contiguous(), wg, wu)
    assert torch.equal(a, b)


def test_gated_linear_shapes_masters_and_frozen_operands():
    from stacr_b200.ops import nn_ops

    x, wg, wu, bg, bu, dh = gated_inputs(2 * 3 * 5, 64, 72)
    x3 = x.view(2, 3, 5, 64)
    assert nn_ops.gated_linear(x3, wg, wu).shape == (2, 3, 5, 72)
    ref = nn_ops.gated_linear(x, wg, wu)
    assert torch.equal(nn_ops.gated_linear(x3, wg, wu).view(-1, 72), ref)
    # fp32 masters and activations under autocast: fp32 gradients from the same products
    masters = [t.float().requires_grad_() for t in (wg, wu)]
    xf = x.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = nn_ops.gated_linear(xf, *masters)
    assert torch.equal(h, ref)
    full = torch.autograd.grad(h, (xf, *masters), dh)
    assert [t.dtype for t in full] == [torch.float32] * 3
    leaves = [x.clone().requires_grad_(), wg.clone().requires_grad_(), wu.clone().requires_grad_()]
    half = torch.autograd.grad(nn_ops.gated_linear(*leaves), leaves, dh)
    for a, b in zip(full, half):
        inside(b, a.double(), a.double().abs() * HALF[torch.bfloat16] + 1e-30)
    # each operand frozen in turn: the others' gradients are the same bits
    for frozen in range(3):
        some = [t.detach().clone().requires_grad_(i != frozen) for i, t in enumerate(leaves)]
        nn_ops.gated_linear(*some).backward(dh)
        assert some[frozen].grad is None
        for i in range(3):
            if i != frozen:
                assert torch.equal(some[i].grad, half[i])
    # one weight in both places
    w = wg.clone().requires_grad_()
    (both,) = torch.autograd.grad(nn_ops.gated_linear(x, w, w), w, dh)
    a, b = wg.clone().requires_grad_(), wg.clone().requires_grad_()
    ga, gb = torch.autograd.grad(nn_ops.gated_linear(x, a, b), (a, b), dh)
    inside(both, (ga + gb).double(), (ga.double().abs() + gb.double().abs()) * 2 * HALF[torch.bfloat16])
    # widths that are no multiple of 8 go through the framework ops
    odd = nn_ops.gated_linear(torch.randn(4, 12, device="cuda").bfloat16(), torch.randn(10, 12, device="cuda").bfloat16(), torch.randn(10, 12, device="cuda").bfloat16())
    assert odd.shape == (4, 10)


def test_gated_linear_uses_lent_gradient_slots():
    from stacr_b200.ops import nn_ops

    x, wg, wu, _, _, dh = gated_inputs(300, 128, 264)
    plain = [t.float().requires_grad_() for t in (wg, wu)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = torch.autograd.grad(nn_ops.gated_linear(x, *plain), plain, dh)
    flat = torch.full((2 * 264 * 128 + 64,), 7.0, device="cuda")
    lent, calls = [torch.nn.Parameter(t.float()) for t in (wg, wu)], []
    for i, p in enumerate(lent):
        p._sb_grad_out, p._sb_grad_fresh = flat[32 + i * 264 * 128:][:264 * 128].view(264, 128), True
        p._sb_grad_ready = lambda i=i: calls.append(i)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        nn_ops.gated_linear(x, *lent).backward(dh)
    assert sorted(calls) == [0, 1] and all(p.grad is None and not p._sb_grad_fresh for p in lent)
    for p, w in zip(lent, want):
        assert torch.equal(p._sb_grad_out, w)
    assert bool((flat[:32] == 7).all() and (flat[-32:] == 7).all())


@pytest.mark.parametrize("recompute", [False, True])
def test_operators_survive_offloaded_saved_tensors(recompute):
    from stacr_b200.ops import nn_ops

    x, wg, wu, _, _, dh = gated_inputs(150, 64, 136)
    inv, _ = nn_ops.rotary_frequencies(64, device="cuda")
    results = []
    for offload in (False, True):
        leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu)]
        with torch.autograd.graph.save_on_cpu(pin_memory=True) if offload else torch.enable_grad():
            h = nn_ops.gated_linear(*leaves, recompute=recompute)
            p = nn_ops.gated_product(leaves[0], leaves[0])
            q, _ = nn_ops.rotary(leaves[0].view(10, 15, 1, 64), None, inv, 3)
        results.append([*torch.autograd.grad(h, leaves, dh), *torch.autograd.grad(p.sum() + q.square().sum(), leaves[0])])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("m", [3, 70])
def test_gated_linear_takes_operands_of_any_alignment_and_order(m):
    from stacr_b200.ops import nn_ops

    tensors = [t for i, t in enumerate(gated_inputs(m, 64, 136)) if i not in (3, 4)]
    want = None
    for move in ("as is", "shifted", "transposed"):
        moved = []
        for t in tensors:
            if move == "shifted":       # two bytes behind a 16-byte boundary
                t = torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)
            elif move == "transposed":
                t = t.t().contiguous().t()
            moved.append(t)
        leaves = [t.detach().requires_grad_() for t in moved[:3]]
        h = nn_ops.gated_linear(*leaves)
        got = [h.detach(), *torch.autograd.grad(h, leaves, moved[3])]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want)), move


def test_gated_linear_nonfinite_values_stay_in_their_rows_and_columns():
    from stacr_b200.ops import nn_ops

    x, wg, wu, _, _, dh = gated_inputs(130, 64, 136)
    for at, value in ((0, float("inf")), (129, float("nan"))):
        bad = x.clone()
        bad[at, 3] = value
        h = nn_ops.gated_linear(bad, wg, wu)
        rows = ~torch.isfinite(h).all(1)
        assert rows[at] and int(rows.sum()) == 1
        clean = torch.ones(130, dtype=torch.bool, device="cuda")
        clean[at] = False
        assert torch.equal(h[clean], nn_ops.gated_linear(x, wg, wu)[clean])
        # and backward: dx is clean in the other rows, whatever lies beyond the matrices' edges in a tile
        leaf = bad.requires_grad_()
        (dx,) = torch.autograd.grad(nn_ops.gated_linear(leaf, wg, wu), leaf, dh)
        assert bool(torch.isfinite(dx[clean]).all())


def test_gated_linear_repeats_bit_for_bit_and_runs_on_a_side_stream():
    from stacr_b200.ops import nn_ops

    x, wg, wu, _, _, dh = gated_inputs(700, 512, 1096)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    runs = []
    side = torch.cuda.Stream()
    for k in range(4):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            h = nn_ops.gated_linear(*leaves, recompute=k >= 2)
            runs.append([h.detach(), *torch.autograd.grad(h, leaves, dh)])
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1])) and all(torch.equal(a, b) for a, b in zip(runs[2], runs[3]))
    assert torch.equal(runs[0][0], runs[2][0])


@pytest.mark.parametrize("recompute", [False, True])
def test_gated_linear_offsets_beyond_32_bits(recompute):
    from stacr_b200.ops import nn_ops

    m, k, f = 270001, 64, 8192          # 2.2e9 features
    x, wg, wu, bg, bu, _ = gated_inputs(m, k, f)
    dh = torch.randn(1, f, device="cuda").bfloat16().expand(m, f)
    xl = x.requires_grad_()
    h = nn_ops.gated_linear(xl, wg, wu, bg, bu, recompute=recompute)
    (dx,) = torch.autograd.grad(h, xl, dh)
    for rows in (slice(0, 40), slice(262140, 262180), slice(m - 40, m)):
        leaves = (x.detach()[rows], wg, wu, bg, bu)
        g, u, want, grads = gated_exact(*leaves, dh[rows], "silu")
        bounds = gated_bounds(*leaves, dh[rows], "silu", g, u, keep=not recompute)
        inside(h.detach()[rows], want, bounds[0], "h")
        inside(dx[rows], grads[0], bounds[1], "dx")


def test_gated_product_sizes_beyond_32_bits():
    from stacr_b200.ops import nn_ops

    n = 2 ** 31 + 9
    gate = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    gate[-5:] = 2.0
    gate[:3] = 1.0
    out = nn_ops.gated_product(gate, gate)
    want = F.silu(torch.tensor([1.0, 2.0], dtype=torch.float64)) * torch.tensor([1.0, 2.0], dtype=torch.float64)
    assert bool((out[:3] == want[0].to(torch.bfloat16).cuda()).all()) and bool((out[-5:] == want[1].to(torch.bfloat16).cuda()).all())
    assert not bool(out[3:-5].any())


def test_two_captured_graphs_replayed_at_once_do_not_disturb_each_other():
    from stacr_b200.ops import nn_ops
    from stacr_b200.optim import clip_grad_norm_

    inv, _ = nn_ops.rotary_frequencies(64, device="cuda")
    jobs = []
    for seed, (m, k, f) in enumerate(((700, 512, 1096), (40, 1024, 2056))):
        x, wg, wu, _, _, dh = gated_inputs(m, k, f, seed=seed)
        leaves = [t.requires_grad_() for t in (x, wg, wu)]
        q = torch.randn(2, 33, 4, 64, device="cuda")
        params = clip_params([(257, 129), (5000,)], (torch.float32,), seed=seed)
        fresh = [p.grad.clone() for p in params]

        def job(leaves=leaves, dh=dh, q=q, params=params, fresh=fresh):
            for p, g in zip(params, fresh):
                p.grad.copy_(g)
            h = nn_ops.gated_linear(*leaves)
            grads = torch.autograd.grad(h, leaves, dh)
            return [h.detach(), *grads, nn_ops.gated_product(q, q + 1), nn_ops.rotary(q, None, inv, 5)[0], clip_grad_norm_(params, 0.3), *(p.grad for p in params)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in job()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = job()
        jobs.append((graph, got, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, stream in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _ in jobs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ gradient norm and clipping
def clip_params(shapes, dtypes, std=1.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dtypes[i % len(dtypes)]))
        p.grad = (torch.randn(s, generator=gen, device="cuda") * std).to(p.dtype)
        params.append(p)
    return params


def check_clip(params, max_norm):
    from stacr_b200.optim import clip_grad_norm_, grad_norm

    before = [p.grad.double() for p in params]
    total = torch.stack([g.square().sum() for g in before]).sum().sqrt()
    # 16 squares summed in fp32 (16 roundings, halved by the root), fp64 beyond, one rounding of the result
    assert abs(float(grad_norm(params)) - float(total)) <= (16 / 2 + 2) * 2.0 ** -24 * float(total)
    norm = clip_grad_norm_(params, max_norm)
    assert abs(float(norm) - float(total)) <= (16 / 2 + 2) * 2.0 ** -24 * float(total)
    factor = min(1.0, max_norm / (float(total) + 1e-6))
    for p, g in zip(params, before):
        if factor == 1.0:
            assert torch.equal(p.grad.double(), g)
        else:      # the factor inherits the norm's roundings and its own, and the product is rounded to the gradient's type
            inside(p.grad, g * factor, g.abs() * factor * (HALF[p.dtype] + 14 * 2.0 ** -24) + TINY[p.dtype])


@pytest.mark.parametrize("max_norm", [1e-3, 0.7, 1e6])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,), (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("shapes", [[(1,)], [(5,), (0,), (3, 7), ()], [(1000, 33), (4096,), (4097,), (16385,)], [(257, 1031)] * 3 + [(17,)] * 40])
def test_clip_grad_norm(shapes, dtypes, max_norm):
    check_clip(clip_params(shapes, dtypes), max_norm)


def test_clip_more_tensors_than_one_table_holds():
    check_clip(clip_params([(3,), (129, 5), (2048,)] * 500, (torch.float32, torch.bfloat16)), 0.5)


def test_clip_values_whose_squares_leave_fp32():
    check_clip(clip_params([(100, 100), (7,)], (torch.float32, torch.bfloat16), std=1e25), 1.0)
    check_clip(clip_params([(100, 100), (7,)], (torch.float32, torch.bfloat16), std=1e-25), 1e-26)
    params = clip_params([(50, 50)], (torch.float32,), std=1e-3)
    params[0].grad[3, 4] = 2e30
    check_clip(params, 1.0)


def test_clip_unaligned_views_transposes_and_canaries():
    buffer = torch.full((5000,), 3.0, device="cuda")
    params = []
    for off, n in ((1, 1001), (1003, 64), (1070, 3000)):
        p = torch.nn.Parameter(torch.empty(n, device="cuda"))
        p.grad = buffer[off:off + n]
        params.append(p)
    t = torch.nn.Parameter(torch.empty(40, 30, device="cuda").t())
    t.grad = torch.randn(40, 30, device="cuda").t()
    params.append(t)
    check_clip(params, 1.0)
    outside = torch.ones(5000, dtype=torch.bool, device="cuda")
    for off, n in ((1, 1001), (1003, 64), (1070, 3000)):
        outside[off:off + n] = False
    assert bool((buffer[outside] == 3.0).all()) and not bool((buffer[~outside] == 3.0).any())


def test_clip_shared_nonfinite_sparse_strided_and_overlapping_gradients():
    from stacr_b200.optim import clip_grad_norm_, grad_norm

    (p,) = clip_params([(64, 64)], (torch.float32,))
    twin = torch.nn.Parameter(torch.empty_like(p))
    twin.grad = p.grad
    before = p.grad.clone()
    norm = clip_grad_norm_([p, twin, p], 1.0)
    inside(p.grad, before.double() / float(before.double().norm()), before.double().abs() / float(before.double().norm()) * 2.0 ** -19)
    assert abs(float(norm) - float(before.double().norm())) < 1e-4
    version = p.grad._version
    clip_grad_norm_((q for q in [p]), 0.5)
    assert p.grad._version > version
    # strided gradients are not one stretch of memory: the framework's function takes them
    s = torch.nn.Parameter(torch.empty(8, 4, device="cuda"))
    s.grad = torch.ones(8, 8, device="cuda")[:, ::2]
    assert abs(float(clip_grad_norm_(s, 1.0)) - 32 ** 0.5) < 1e-5 and abs(float(s.grad.norm()) - 1) < 1e-5
    # part of one gradient inside another
    flat = torch.ones(100, device="cuda")
    a, b = torch.nn.Parameter(torch.empty(60, device="cuda")), torch.nn.Parameter(torch.empty(60, device="cuda"))
    a.grad, b.grad = flat[:60], flat[40:]
    with pytest.raises(ValueError):
        clip_grad_norm_([a, b], 1.0)
    assert bool((flat == 1).all())
    # infinities and NaN: the norm says so, an error is raised on request before anything is scaled
    for value in (float("inf"), float("nan")):
        (p,) = clip_params([(1000,)], (torch.float32,))
        p.grad[500] = value
        kept = p.grad.clone()
        with pytest.raises(RuntimeError):
            clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert torch.equal(p.grad.nan_to_num(5, 6), kept.nan_to_num(5, 6))
        assert not torch.isfinite(grad_norm(p))
        want = torch.nn.Parameter(torch.empty_like(p))
        want.grad = kept
        torch.nn.utils.clip_grad_norm_(want, 1.0)
        clip_grad_norm_(p, 1.0)
        assert torch.equal(p.grad.nan_to_num(5, 6), want.grad.nan_to_num(5, 6))
    zero = torch.nn.Parameter(torch.empty(10, device="cuda"))
    zero.grad = torch.zeros(10, device="cuda")
    assert float(clip_grad_norm_(zero, 1.0)) == 0.0
    empty = torch.nn.Parameter(torch.empty(0, 3, device="cuda"))
    empty.grad = torch.empty(0, 3, device="cuda")
    assert float(clip_grad_norm_(empty, 1.0)) == 0.0


def test_clip_repeats_bit_for_bit():
    from stacr_b200.optim import clip_grad_norm_

    results = []
    for _ in range(3):
        params = clip_params([(1111, 777), (33,), (2049,)], (torch.float32, torch.bfloat16), seed=5)
        results.append([clip_grad_norm_(params, 0.3), *(p.grad for p in params)])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


def test_clip_sizes_beyond_32_bits():
    from stacr_b200.optim import clip_grad_norm_

    p = torch.nn.Parameter(torch.empty(2 ** 32 + 3, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    p.grad[:2] = 3.0
    p.grad[-2:] = 4.0
    norm = clip_grad_norm_(p, 1.0)
    assert abs(float(norm) - 50 ** 0.5) < 1e-5
    assert abs(float(p.grad[-1]) - 4 / 50 ** 0.5) < 4 / 50 ** 0.5 * 2.0 ** -8 and float(p.grad[2 ** 31]) == 0.0


# ------------------------------------------------------------------------------------------------ together
def unfused(model):
    """The same model with its projections hooked, so that gate, up and their product run as separate layers."""
    return [m.register_forward_hook(lambda *_: None) for name, m in model.named_modules() if name.endswith("gate_proj")]


@pytest.mark.parametrize("recompute", [False, True])
def test_llama_step_with_the_fused_block_tracks_fp32(recompute):
    from stacr_b200.models import build_model
    from stacr_b200.optim import clip_grad_norm_

    torch.manual_seed(0)
    model = build_model("llama-tiny", mlp_recompute=recompute).cuda()
    ids = torch.randint(0, 1024, (3, 77), device="cuda")
    model(input_ids=ids, labels=ids).loss.backward()           # fp32: framework GEMMs, the same rotary kernel
    want = {n: p.grad.clone() for n, p in model.named_parameters()}

    def step():
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    fused = step()
    handles = unfused(model)
    separate = step()
    for h in handles:
        h.remove()
    err = {n: [float((g[n] - want[n]).norm() / want[n].norm()) for g in (fused, separate)] for n in want}
    # the fused block rounds less often than the separate layers: its gradients are no further from the fp32 step's, within a quarter
    assert all(a <= 1.25 * b + 1e-4 for a, b in err.values()), err
    total = torch.stack([g.double().square().sum() for g in separate.values()]).sum().sqrt()
    norm = clip_grad_norm_(model.parameters(), 0.1)
    assert abs(float(norm) - float(total)) <= (16 / 2 + 2) * 2.0 ** -24 * float(total)
    after = torch.stack([p.grad.double().square().sum() for p in model.parameters()]).sum().sqrt()
    assert abs(float(after) - 0.1) < 1e-6


def test_llama_under_saved_tensor_hooks_saves_what_separate_layers_save():
    from stacr_b200.models import build_model

    torch.manual_seed(0)
    model = build_model("llama-tiny").cuda()
    ids = torch.randint(0, 1024, (1, 40), device="cuda")
    saved = []
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        model(input_ids=ids, labels=ids).loss.backward()
    assert not any(t.dtype == torch.uint8 for t in saved)
    # gate, its activation and up in each of the two layers, and the down projection's input
    assert sum(t.dtype == torch.bfloat16 and t.shape[-1] == 688 and t.numel() == 40 * 688 for t in saved) >= 8


def test_llama_mlp_with_compressed_projections_runs_the_gated_product():
    import stacr_b200 as S
    from stacr_b200.models import build_model
    from stacr_b200.ops import nn_kernels

    torch.manual_seed(0)
    model = build_model("llama-tiny").cuda()
    layers = S.apply_stacr(model, rank=8, residual_budget=0.01, surface="mlp", min_features=64)
    S.set_step(layers, 0)
    mlp = model.model.layers[0].mlp
    x = torch.randn(2, 64, 256, device="cuda").bfloat16()          # the basis kernels take multiples of 8 rows
    calls = []
    real = nn_kernels.gated_product_fwd
    nn_kernels.gated_product_fwd = lambda *a: calls.append(1) or real(*a)
    try:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = mlp(x)
            assert len(calls) == 1
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
                z = mlp(x)                     # the activation and the product as two ops
            assert len(calls) == 1
            gate, up = mlp.gate_proj(x).double(), mlp.up_proj(x).double()
    finally:
        nn_kernels.gated_product_fwd = real
    # h is rounded once here and twice there, so the two differ by three half steps of it at most, each output by one more
    h, w, e = (F.silu(gate) * up).abs().detach(), mlp.down_proj.weight.detach().to(torch.bfloat16).double().abs(), HALF[torch.bfloat16]
    inside(y.detach(), z.detach().double(), 3 * e * (1 + e) * (h @ w.t()) + 2 * e * z.detach().double().abs() + 1e-6)
    y.float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in mlp.parameters() if p.grad is not None)


def test_llama_step_replayed_from_a_cuda_graph_equals_the_eager_step():
    from stacr_b200.models import build_model
    from stacr_b200.optim import clip_grad_norm_

    torch.manual_seed(0)
    model = build_model("llama-tiny", rope_scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64)).cuda()
    params = list(model.parameters())
    for p in params:
        p.grad = torch.zeros_like(p)

    def step(ids):
        for p in params:
            p.grad.zero_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        return loss.detach(), clip_grad_norm_(params, 0.05)

    batches = [torch.randint(0, 1024, (2, 65), device="cuda") for _ in range(3)]
    static = batches[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, norm = step(static)
    for ids in batches[1:] + batches[:1]:
        static.copy_(ids)
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone(), norm.clone()] + [p.grad.clone() for p in params]
        again_loss, again_norm = step(ids)
        # the embedding's gradient is summed with atomics, whose order may differ: equality up to their roundings
        assert torch.equal(got[0], again_loss)
        torch.testing.assert_close(got[1], again_norm, rtol=1e-5, atol=0)
        for a, p in zip(got[2:], params):
            torch.testing.assert_close(a, p.grad, rtol=1e-4, atol=1e-7)


def test_neox_with_an_uneven_rotary_part_tracks_fp32():
    from stacr_b200.models import build_model

    torch.manual_seed(0)
    model = build_model("pythia-70m", hidden_size=320, num_hidden_layers=2, num_attention_heads=4, intermediate_size=640, vocab_size=512).cuda()
    assert model.gpt_neox.layers[0].attention.rot == 20
    ids = torch.randint(0, 512, (2, 50), device="cuda")
    with torch.no_grad():
        want = model.double()(input_ids=ids).logits
        model.float()
        got = model(input_ids=ids).logits
    # fp32 layers of width 320 to 640 and depth 2 against fp64
    torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-4)
