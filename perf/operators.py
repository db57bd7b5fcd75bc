"""Workloads of the training step's gated feed-forward, rotary and gradient-clipping operators, with their plain forms.

``run`` computes an operator in elementary torch operations in 32 bits (64 where 32 lose what matters), or, where ``own`` is
true, through the framework's entry points.  ``exact`` restates the operator's definition in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through the feed-forward block of a 1B decoder: the latency of generation, bound by the weights' bytes
        dict(name="gated_token", op="gated", m=1, k=2048, f=8192, act="silu", mode="infer"),
        # a ragged batch of single tokens on another decoder's sizes
        dict(name="gated_tokens_33", op="gated", m=33, k=1536, f=8960, act="silu", mode="infer"),
        # the smallest training step of the test model: two sequences of 127 tokens
        dict(name="gated_train_tiny", op="gated", m=254, k=256, f=688, act="silu", mode="train"),
        # an ordinary training step, forward and backward: 4 x 2048 tokens
        dict(name="gated_train", op="gated", m=8192, k=2048, f=8192, act="silu", mode="train"),
        # an 8B decoder's block with the projections recomputed in the backward pass instead of kept; a ragged token count
        dict(name="gated_train_recompute", op="gated", m=4095, k=4096, f=14336, act="silu", mode="recompute"),
        # the product behind compressed projections, forward and backward, over one training batch
        dict(name="product_train", op="product", m=8192, f=8192, act="silu", dtype="bf16", split=False, mode="train"),
        # odd width, the two halves of one fused projection, 32-bit values
        dict(name="product_odd_halves", op="product", m=333, f=1003, act="gelu_tanh", dtype="fp32", split=True, mode="train"),
        # 64 sequences generating one token each, every one at a far position of its own
        dict(name="rotary_tokens", op="rotary", b=64, s=1, hq=32, hk=8, d=64, rot=64, layout="half", dtype="bf16", positions="each", factor=8.0,
             scale=1.0, mode="infer"),
        # forward and backward of one training batch with grouped key heads
        dict(name="rotary_train", op="rotary", b=4, s=2048, hq=32, hk=8, d=128, rot=128, layout="half", dtype="bf16", positions="row", factor=1.0,
             scale=1.0, mode="train"),
        # a long context: a quarter of each head, pairs side by side, stretched frequencies and scaled scores
        dict(name="rotary_long_partial", op="rotary", b=1, s=30011, hq=32, hk=32, d=80, rot=20, layout="interleaved", dtype="fp16", positions="each",
             factor=16.0, scale=1.277, mode="train"),
        # clipping the gradients of the test model
        dict(name="clip_tiny", op="clip", layers=2, hidden=256, kv=128, ffn=688, vocab=1024, dtype="fp32", clips=True),
        # clipping the gradients of a 1B decoder
        dict(name="clip_1b", op="clip", layers=16, hidden=2048, kv=512, ffn=8192, vocab=128256, dtype="fp32", clips=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gated", "product", "rotary", "clip"))
    if op == "gated":
        k, f = 8 * _log(rng, 16, 512), 8 * _log(rng, 32, 1792)
        mode = rng.choice(("infer", "infer", "train", "recompute"))
        m = _log(rng, 1, 8192)
        m = max(1, min(m, 4095 * 4096 * 14336 // (k * f)))
        return dict(op=op, m=m, k=k, f=f, act=rng.choice(("silu", "silu", "gelu", "gelu_tanh")), mode=mode)
    if op == "product":
        m, f = _log(rng, 1, 8192), _log(rng, 100, 8192)
        return dict(op=op, m=m, f=f, act=rng.choice(("silu", "gelu", "gelu_tanh")), dtype=rng.choice(tuple(DTYPES)), split=rng.random() < 0.5,
                    mode=rng.choice(("infer", "train")))
    if op == "rotary":
        d = rng.choice((64, 80, 96, 128))
        rot = rng.choice((d, d, d // 2, d // 4))
        hq = rng.choice((4, 12, 28, 32))
        hk = hq // rng.choice((1, 4))
        s = _log(rng, 1, 30000)
        b = max(1, min(_log(rng, 1, 64), 30000 * 64 // (s * hq)))
        return dict(op=op, b=b, s=s, hq=hq, hk=hk, d=d, rot=rot, layout=rng.choice(("half", "interleaved")), dtype=rng.choice(tuple(DTYPES)),
                    positions=rng.choice(("row", "each")), factor=rng.choice((1.0, 4.0, 16.0)), scale=rng.choice((1.0, 1.139)),
                    mode=rng.choice(("infer", "train")))
    hidden = _log(rng, 64, 2048)
    return dict(op=op, layers=rng.randint(1, 16), hidden=hidden, kv=max(1, hidden // rng.choice((1, 2, 4))), ffn=_log(rng, 128, 8192),
                vocab=_log(rng, 500, 64000), dtype=rng.choice(tuple(DTYPES)), clips=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(shape, gen, std, dtype):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * std).to(dtype)


def _grad_shapes(c):
    """The parameters of a decoder: per layer two norms, q, k, v, o, gate, up, down; then the table and the last norm."""
    h, kv, f = c["hidden"], c["kv"], c["ffn"]
    layer = [(h,), (h,), (h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f)]
    return layer * c["layers"] + [(c["vocab"], h), (h,)]


def _inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if c["op"] == "gated":
        m, k, f, bf = c["m"], c["k"], c["f"], torch.bfloat16
        t = dict(x=_normal((m, k), gen, 1.0, bf), wg=_normal((f, k), gen, 0.02, bf), wu=_normal((f, k), gen, 0.02, bf))
        if c["mode"] != "infer":
            t["dh"] = _normal((m, f), gen, 1e-3, bf)
        return t
    if c["op"] == "product":
        dt, m, f = DTYPES[c["dtype"]], c["m"], c["f"]
        gate_up = _normal((m, 2 * f), gen, 1.5, dt)
        gate, up = gate_up[:, :f], gate_up[:, f:]
        t = dict(gate=gate if c["split"] else gate.contiguous(), up=up if c["split"] else up.contiguous())
        if c["mode"] != "infer":
            t["dout"] = _normal((m, f), gen, 0.1, dt)
        return t
    if c["op"] == "rotary":
        dt, b, s = DTYPES[c["dtype"]], c["b"], c["s"]
        t = dict(q=_normal((b, s, c["hq"], c["d"]), gen, 1.0, dt), k=_normal((b, s, c["hk"], c["d"]), gen, 1.0, dt))
        base = 10000.0 * c["factor"] ** (c["rot"] / max(1, c["rot"] - 2))      # frequencies stretched to a longer context
        t["inv_freq"] = base ** -(torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
        if c["positions"] == "each":       # every sequence starts at a far place of its own
            start = torch.randint(0, 100000, (b, 1), generator=gen, device=DEV)
            t["positions"] = start + torch.arange(s, device=DEV)
        if c["mode"] != "infer":
            t["dq"], t["dk"] = _normal(t["q"].shape, gen, 0.1, dt), _normal(t["k"].shape, gen, 0.1, dt)
        return t
    dt = DTYPES[c["dtype"]]
    sizes = [math.prod(s) for s in _grad_shapes(c)]
    slots = [-(-n // 4) * 4 for n in sizes]
    flat = torch.empty(sum(slots), device=DEV, dtype=dt)
    std = 1e-2
    parts = flat.split(1 << 26)
    [p.copy_(torch.randn(p.shape, generator=gen, device=DEV) * std) for p in parts]
    views = [v[:n] for v, n in zip(flat.split(slots), sizes)]
    [v[n:].zero_() for v, n in zip(flat.split(slots), sizes)]
    return dict(flat=flat, views=views, bound=(0.3 if c["clips"] else 3.0) * std * math.sqrt(sum(sizes)))


def prepare(case, seed):
    t = _inputs(case, seed)
    t["case"] = case
    if case["op"] == "clip":
        # the gradients lie in one buffer, as the data-parallel synchroniser keeps them
        t["params"] = [torch.nn.Parameter(torch.empty(s, device=DEV, dtype=t["flat"].dtype)) for s in _grad_shapes(case)]
        for p, v in zip(t["params"], t["views"]):
            p.grad = v.view(p.shape)
    if case["mode" if "mode" in case else "op"] in ("train", "recompute"):
        for name in ("x", "wg", "wu", "gate", "up", "q", "k"):
            if name in t:
                t[name] = t[name].detach().requires_grad_()
    return t


def _next_bound(state):
    """Every step's bound lies a little below the last one's, so that a pass over gradients that were clipped before still clips."""
    state["bound"] *= 0.9999
    return state["bound"]


# ------------------------------------------------------------------------------------------------ the plain forms
def _act(g, act):
    """(act(g), act'(g))"""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


@torch.no_grad()
def _plain_gated(t, c):
    x, wg, wu = t["x"].float(), t["wg"].float(), t["wu"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, c["act"])
    h = (a * u).bfloat16()
    if c["mode"] == "infer":
        return h
    dh = t["dh"].float()
    dg, du = dh * u * da, dh * a
    return [h] + [r.bfloat16() for r in (dg @ wg + du @ wu, dg.T @ x, du.T @ x)]


@torch.no_grad()
def _plain_product(t, c):
    gate, up, dt = t["gate"].float(), t["up"].float(), t["gate"].dtype
    a, da = _act(gate, c["act"])
    out = (a * up).to(dt)
    if c["mode"] == "infer":
        return out
    d = t["dout"].float()
    return [out, (d * up * da).to(dt), (d * a).to(dt)]


def _rotate(x, cos, sin, c):
    rot, y = c["rot"], x.float()
    r, rest = y[..., :rot], y[..., rot:]
    if c["layout"] == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((r, rest), -1).to(x.dtype)


def _positions(t, c):
    return t["positions"] if "positions" in t else torch.arange(c["s"], device=DEV)[None]


@torch.no_grad()
def _plain_rotary(t, c):
    angle = (_positions(t, c).double()[..., None] * t["inv_freq"])[:, :, None]
    cos, sin = (c["scale"] * angle.cos()).float(), (c["scale"] * angle.sin()).float()
    out = [_rotate(t["q"], cos, sin, c), _rotate(t["k"], cos, sin, c)]
    if c["mode"] == "infer":
        return out
    return out + [_rotate(t["dq"], cos, -sin, c), _rotate(t["dk"], cos, -sin, c)]


@torch.no_grad()
def _plain_clip(t, c):
    bound, flat = _next_bound(t), t["flat"]
    norm = flat.double().square().sum().sqrt()
    flat.copy_(flat.float() * (bound / (norm + 1e-6)).clamp(max=1.0).float())
    return norm.float(), flat


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_gated(t, c):
    from stacr_b200.ops import nn_ops

    if c["mode"] == "infer":
        with torch.no_grad():
            return nn_ops.gated_linear(t["x"], t["wg"], t["wu"], activation=c["act"])
    h = nn_ops.gated_linear(t["x"], t["wg"], t["wu"], activation=c["act"], recompute=c["mode"] == "recompute")
    return [h, *torch.autograd.grad(h, (t["x"], t["wg"], t["wu"]), t["dh"])]


def _own_product(t, c):
    from stacr_b200.ops import nn_ops

    if c["mode"] == "infer":
        with torch.no_grad():
            return nn_ops.gated_product(t["gate"], t["up"], activation=c["act"])
    out = nn_ops.gated_product(t["gate"], t["up"], activation=c["act"])
    return [out, *torch.autograd.grad(out, (t["gate"], t["up"]), t["dout"])]


def _own_rotary(t, c):
    from stacr_b200.ops import nn_ops

    def rotated():
        return nn_ops.rotary(t["q"], t["k"], t["inv_freq"], t.get("positions"), interleaved=c["layout"] == "interleaved", scale=c["scale"])

    if c["mode"] == "infer":
        with torch.no_grad():
            return list(rotated())
    q, k = rotated()
    return [q, k, *torch.autograd.grad((q, k), (t["q"], t["k"]), (t["dq"], t["dk"]))]


def _own_clip(t, c):
    from stacr_b200.optim import clip_grad_norm_

    return clip_grad_norm_(t["params"], _next_bound(t)), t["flat"]


def run(state):
    c = state["case"]
    if own:
        return {"gated": _own_gated, "product": _own_product, "rotary": _own_rotary, "clip": _own_clip}[c["op"]](state, c)
    return {"gated": _plain_gated, "product": _plain_product, "rotary": _plain_rotary, "clip": _plain_clip}[c["op"]](state, c)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "gated":
        mk, kf, mf = c["m"] * c["k"], c["k"] * c["f"], c["m"] * c["f"]
        if c["mode"] == "infer":
            return {"bytes": 2 * (mk + 2 * kf + mf), "flops": 4 * mk * c["f"]}
        # x, both weights, dh in; h, dx, both dW out; two products forward and four backward (a recomputed pair is not counted)
        return {"bytes": 2 * (2 * mk + 4 * kf + 2 * mf), "flops": 12 * mk * c["f"]}
    if c["op"] == "product":
        n, size = c["m"] * c["f"], DTYPES[c["dtype"]].itemsize
        return {"bytes": (3 if c["mode"] == "infer" else 6) * n * size, "flops": (6 if c["mode"] == "infer" else 18) * n}
    if c["op"] == "rotary":
        n = c["b"] * c["s"] * (c["hq"] + c["hk"])
        passes = 1 if c["mode"] == "infer" else 2
        return {"bytes": passes * 2 * n * c["d"] * DTYPES[c["dtype"]].itemsize, "flops": passes * 3 * n * c["rot"]}
    n = sum(math.prod(s) for s in _grad_shapes(c))
    return {"bytes": (2 if c["clips"] else 1) * n * DTYPES[c["dtype"]].itemsize, "flops": (3 if c["clips"] else 2) * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c, t = case, _inputs(case, seed)
    F = torch.nn.functional
    f = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}
    if c["op"] == "gated":
        train = c["mode"] != "infer"
        x, wg, wu = (t.pop(n).double().requires_grad_(train) for n in ("x", "wg", "wu"))
        h = f[c["act"]](F.linear(x, wg)) * F.linear(x, wu)
        return [h.detach(), *torch.autograd.grad(h, (x, wg, wu), t["dh"].double())] if train else h
    if c["op"] == "product":
        train = c["mode"] != "infer"
        gate, up = (t[n].double().requires_grad_(train) for n in ("gate", "up"))
        out = f[c["act"]](gate) * up
        return [out.detach(), *torch.autograd.grad(out, (gate, up), t["dout"].double())] if train else out
    if c["op"] == "rotary":
        theta = torch.einsum("bs,j->bsj", _positions(t, c).double(), t["inv_freq"]).unsqueeze(2)
        turn = torch.polar(torch.full_like(theta, c["scale"]), theta)

        def turned(v, by):
            v = v.double()
            head = v[..., :c["rot"]].unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" else v[..., :c["rot"]].unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * by)
            z = z.transpose(-1, -2) if c["layout"] == "half" else z
            return torch.cat((z.flatten(-2), v[..., c["rot"]:]), -1)

        out = [turned(t["q"], turn), turned(t["k"], turn)]
        return out if c["mode"] == "infer" else out + [turned(t["dq"], turn.conj()), turned(t["dk"], turn.conj())]
    total = torch.stack([v.double().pow(2).sum() for v in t["views"]]).sum().sqrt()
    bound = t["bound"] * 0.9999
    return total, t["flat"].double() * min(1.0, bound / (float(total) + 1e-6))
