"""Rotary positions, gated feed-forward and gradient clipping off the GPU: the framework-op forms, frequency scalings and refusals."""

import math

import pytest
import torch
from torch.nn import functional as F

from stacr_b200.models import build_model
from stacr_b200.ops import nn_ops
from stacr_b200.optim import clip_grad_norm_, grad_norm

HALF_STEP = 2.0 ** -24      # largest relative error of one fp32 rounding


def turned(x, positions, inv, interleaved, scale=1.0):
    """The definition in 64 bits, by complex multiplication."""
    x, rot = x.double(), 2 * inv.numel()
    theta = positions.double()[..., None] * inv
    head = x[..., :rot].unflatten(-1, (-1, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(head.contiguous()) * torch.polar(torch.full_like(theta, scale), theta)[:, :, None]
    z = torch.view_as_real(z)
    return torch.cat(((z if interleaved else z.transpose(-1, -2)).flatten(-2), x[..., rot:]), -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot,d", [(16, 16), (6, 20), (2, 2)])
def test_rotary_framework_form_is_the_rotation(interleaved, rot, d):
    torch.manual_seed(0)
    inv, _ = nn_ops.rotary_frequencies(rot)
    q, k = torch.randn(2, 5, 4, d, requires_grad=True), torch.randn(2, 5, 2, d)
    pos = torch.tensor([[0, 1, 2, 3, 4], [99990, 7, 7, 12, 5]])
    q2, k2 = nn_ops.rotary(q, k, inv, pos, interleaved=interleaved, scale=1.25)
    # cos and sin rounded, two products and a sum: at most 4 roundings of values bounded by 1.25 (|a| + |b|)
    tol = 4 * HALF_STEP * 1.25 * 2 * float(max(q.abs().max(), k.abs().max()))
    assert float((q2.double() - turned(q, pos, inv, interleaved, 1.25)).abs().max()) <= tol
    assert float((k2.double() - turned(k, pos, inv, interleaved, 1.25)).abs().max()) <= tol
    g = torch.randn_like(q2)
    (dq,) = torch.autograd.grad(q2, q, g)
    assert float((dq.double() - turned(g, -pos, inv, interleaved, 1.25)).abs().max()) <= 4 * HALF_STEP * 1.25 * 2 * float(g.abs().max())


def test_rotary_positions_forms_agree():
    inv, _ = nn_ops.rotary_frequencies(8)
    q = torch.randn(2, 3, 1, 8)
    base = nn_ops.rotary(q, None, inv)[0]
    for pos in (torch.arange(3), torch.arange(3, dtype=torch.int32)[None], torch.arange(3).expand(2, 3), torch.arange(3, dtype=torch.int16)):
        assert torch.equal(nn_ops.rotary(q, None, inv, pos)[0], base)
    assert torch.equal(nn_ops.rotary(q, None, inv, 5)[0], nn_ops.rotary(q, None, inv, torch.arange(5, 8))[0])
    assert torch.equal(nn_ops.rotary(q, None, inv, torch.tensor([[4], [9]]))[0][1], nn_ops.rotary(q[1:], None, inv, torch.full((1, 3), 9))[0][0])


def test_rotary_of_nothing():
    inv, _ = nn_ops.rotary_frequencies(8)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        q, k = nn_ops.rotary(torch.zeros(shape), torch.zeros(shape), inv)
        assert q.shape == k.shape == shape


def test_rotary_refusals():
    inv, _ = nn_ops.rotary_frequencies(8)
    q, k = torch.randn(2, 3, 4, 8), torch.randn(2, 3, 2, 8)
    for bad in (q[0], torch.randn(2, 4, 2, 8), torch.randn(1, 3, 2, 8), torch.randn(2, 3, 2, 6), k.double()):
        with pytest.raises(ValueError):
            nn_ops.rotary(q, bad, inv)
    with pytest.raises(ValueError):
        nn_ops.rotary(q[0], None, inv)
    with pytest.raises(TypeError):
        nn_ops.rotary(q.long(), None, inv)
    for bad in (inv[None], torch.ones(5), torch.ones(0), torch.ones(4, dtype=torch.int64)):
        with pytest.raises(ValueError):
            nn_ops.rotary(q, k, bad)
    for bad in (torch.zeros(2), torch.zeros(4).long(), torch.zeros(3, 3).long(), torch.zeros(1, 2, 3).long()):
        with pytest.raises((ValueError, TypeError)):
            nn_ops.rotary(q, k, inv, bad)
    with pytest.raises(TypeError):
        nn_ops.rotary(q, k, inv, torch.zeros(3))


def test_rotary_frequency_scalings():
    dim, base = 64, 10000.0
    plain, one = nn_ops.rotary_frequencies(dim, base)
    assert one == 1.0 and plain.dtype == torch.float64 and float(plain[0]) == 1.0
    assert math.isclose(float(plain[-1]), base ** -(62 / 64), rel_tol=1e-14)
    assert torch.equal(nn_ops.rotary_frequencies(dim, base, {"type": "linear", "factor": 4.0})[0], plain / 4)
    ntk = nn_ops.rotary_frequencies(dim, base, {"rope_type": "ntk", "factor": 4.0})[0]
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(plain[-1]) / 4, rel_tol=1e-12)
    dyn = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=1024)
    assert torch.equal(nn_ops.rotary_frequencies(dim, base, dyn, seq_len=1024)[0], plain)
    assert math.isclose(float(nn_ops.rotary_frequencies(dim, base, dyn, seq_len=4096)[0][-1]), float(plain[-1]) / 7, rel_tol=1e-12)
    original = 2048
    turns = original * plain / (2 * math.pi)
    yarn, scale = nn_ops.rotary_frequencies(dim, base, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=original))
    assert math.isclose(scale, 0.1 * math.log(8) + 1)
    # one pair of slack at either end of the blend: its ends are rounded to whole pairs
    kept, divided = (turns > 32 * base ** (2 / dim)), (turns < base ** (-2 / dim))
    assert torch.allclose(yarn[kept], plain[kept], rtol=1e-12) and torch.allclose(yarn[divided], plain[divided] / 8, rtol=1e-12)
    assert bool((yarn <= plain * (1 + 1e-12)).all() and (yarn >= plain / 8 * (1 - 1e-12)).all())
    l3 = nn_ops.rotary_frequencies(dim, base, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                   original_max_position_embeddings=original))[0]
    assert torch.equal(l3[turns >= 4], plain[turns >= 4]) and torch.equal(l3[turns <= 1], plain[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert bool(mid.any()) and bool(((l3[mid] < plain[mid]) & (l3[mid] > plain[mid] / 8)).all())


@pytest.mark.parametrize("dim,base,scaling", [
    (7, 1e4, None), (0, 1e4, None), (8, -1.0, None), (8, 1e4, {"rope_type": "spiral", "factor": 2}), (8, 1e4, {"type": "linear"}),
    (8, 1e4, {"type": "linear", "factor": 0.5}), (8, 1e4, {"type": "yarn", "factor": 2}),
    (8, 1.0, {"type": "yarn", "factor": 2, "original_max_position_embeddings": 64}),
    (8, 1e4, {"type": "llama3", "factor": 2, "original_max_position_embeddings": 64, "low_freq_factor": 4, "high_freq_factor": 4})])
def test_rotary_frequency_refusals(dim, base, scaling):
    with pytest.raises(ValueError):
        nn_ops.rotary_frequencies(dim, base, scaling)


def test_gated_framework_forms_and_refusals():
    torch.manual_seed(0)
    x, wg, wu = torch.randn(3, 5, 16), torch.randn(24, 16), torch.randn(24, 16)
    for name, act in (("silu", F.silu), ("gelu", F.gelu), ("gelu_tanh", lambda t: F.gelu(t, approximate="tanh"))):
        assert torch.equal(nn_ops.gated_linear(x, wg, wu, activation=name), act(F.linear(x, wg)) * F.linear(x, wu))
        assert torch.equal(nn_ops.gated_product(x, x + 1, name), act(x) * (x + 1))
    assert nn_ops.gated_linear(x[:0], wg, wu).shape == (0, 5, 24)
    for call in (lambda: nn_ops.gated_product(x, x[:1]), lambda: nn_ops.gated_product(x, x, "relu6"), lambda: nn_ops.gated_linear(x, wg, wu[:8]),
                 lambda: nn_ops.gated_linear(x[..., :8], wg, wu), lambda: nn_ops.gated_linear(x, wg, wu, torch.zeros(16)),
                 lambda: nn_ops.gated_linear(x, wg, wu, activation="swish2"), lambda: nn_ops.gated_linear(x, wg[0], wu[0])):
        with pytest.raises(ValueError):
            call()


def test_clipping_follows_the_framework_function_on_the_cpu():
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s)) for s in ((3, 5), (7,), ())] + [torch.nn.Parameter(torch.zeros(2))]
    for p in params[:-1]:
        p.grad = torch.randn_like(p)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, t in zip(params[:-1], twin):
        t.grad = p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(twin, 0.5)
    assert torch.equal(grad_norm(params), want)
    assert torch.equal(clip_grad_norm_((p for p in params), 0.5), want)
    assert all(torch.equal(p.grad, t.grad) for p, t in zip(params[:-1], twin[:-1]))
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    params[0].grad[0, 0] = float("inf")
    with pytest.raises(RuntimeError):
        clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert float(clip_grad_norm_(params[1], 1.0, norm_type=float("inf"))) == float(params[1].grad.abs().max())


def test_llama_scaled_positions_change_the_model_and_default_ones_do_not():
    torch.manual_seed(0)
    ids = torch.randint(0, 1024, (2, 33))
    plain = build_model("llama-tiny")
    scaled = build_model("llama-tiny", rope_scaling={"rope_type": "linear", "factor": 4.0})
    named = build_model("llama-tiny", rope_scaling={"rope_type": "default"})
    for m in (scaled, named):
        m.load_state_dict(plain.state_dict())
    with torch.no_grad():
        a, b, c = (m(input_ids=ids).logits for m in (plain, scaled, named))
    assert float((a - b).abs().max()) > 1e-3
    # angles of 33 positions differ by 33 2^-24 radians between the two forms
    torch.testing.assert_close(a, c, rtol=1e-4, atol=1e-4)


# ---- csrc/gated_gemm.cu restated on the host: how reductions are shared among CTA pairs, and in which order tiles are taken
def shares(tiles, num_kb, sms):
    pairs = max(1, sms // 2)
    last = tiles % pairs
    if last == 0:
        return tiles, 1
    splits = min(pairs // last, num_kb // 8)
    if splits < 2:
        return tiles, 1
    per = -(-num_kb // splits)
    splits = -(-num_kb // per)
    return (tiles, 1) if num_kb - per < 24 else (tiles - last, splits)


@pytest.mark.parametrize("sms", [148, 132, 5, 2, 1])
def test_split_reductions_cover_every_block_once_and_fit_one_round(sms):
    for tiles in (1, 2, 7, 16, 37, 73, 74, 75, 256, 300, 1792):
        for num_kb in (1, 2, 8, 23, 32, 33, 64, 127, 256, 449):
            whole, splits = shares(tiles, num_kb, sms)
            pairs, per, covered = max(1, sms // 2), -(-num_kb // splits), {}
            parts = 0
            for u in range(whole + (tiles - whole) * splits):
                if u < whole:
                    tile, lo, hi = u, 0, num_kb
                else:
                    v = u - whole
                    tile, k = whole + v // splits, v % splits
                    lo, hi = k * per, min((k + 1) * per, num_kb)
                    assert v == parts
                    parts += 1
                assert lo < hi, "a part without blocks would leave its sums unwritten"
                covered.setdefault(tile, []).extend(range(lo, hi))
            assert all(covered[t] == list(range(num_kb)) for t in range(tiles)) and len(covered) == tiles
            assert parts <= pairs and (whole % pairs == 0 or whole == tiles)


@pytest.mark.parametrize("rows", [4, 16])
def test_tile_order_visits_every_tile_once(rows):
    for num_m, num_n in ((1, 1), (3, 7), (4, 5), (17, 3), (32, 64), (33, 2)):
        seen = set()
        for tile in range(num_m * num_n):
            first = tile // (rows * num_n) * rows
            height, r = min(rows, num_m - first), tile % (rows * num_n)
            seen.add((first + r % height, r // height))
        assert seen == {(m, n) for m in range(num_m) for n in range(num_n)}


def test_factors_cut_to_24_bits_join_to_the_value_within_a_step():
    v = torch.cat((torch.randn(4096), torch.tensor([0.0, -0.0, 1e-38, 3e38, float("inf"), -float("inf")])))
    bits = v.view(torch.int32)
    hi, lo = (bits >> 16) & 0xffff, (bits >> 8) & 0xff
    joined = ((hi << 16) | (lo << 8)).to(torch.int32).view(torch.float32)
    finite = torch.isfinite(v)
    assert torch.equal(joined[~finite], v[~finite])
    # cutting takes less than 2^8 of the last mantissa unit: 2^-15 relative, and 2^8 2^-149 among the subnormal values
    assert bool(((joined.double() - v.double()).abs()[finite] <= v.double().abs()[finite] * 2.0 ** -15 + 2.0 ** -141).all())
    assert bool(torch.tensor([0x7fffff00], dtype=torch.int32).view(torch.float32).isnan())      # what arithmetic's NaN is cut to


def test_is_plain_linear_sees_wrapped_and_hooked_layers():
    from stacr_b200.models.common import Linear, is_plain_linear

    layer = Linear(8, 8)
    assert is_plain_linear(layer) and not is_plain_linear(torch.nn.Linear(8, 8))
    handle = layer.register_forward_hook(lambda *_: None)
    assert not is_plain_linear(layer)
    handle.remove()
    assert is_plain_linear(layer)
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *_: None)
    assert not is_plain_linear(layer)
    handle.remove()
    assert is_plain_linear(layer)
    layer.forward = lambda x: x
    assert not is_plain_linear(layer)
