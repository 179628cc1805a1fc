"""More operators of a learned head over splats or tokens, as cases to be timed and compared.

  op       one pass
  norm     between two blocks: the norm after one, its gate, the residual scale and sum, and the norm before the next:
           y = r + s g(G) norm(x), n = norm(y); with `train` also the gradients of x, r, the gate and both weights
  pack     a matrix to 4 bits with a scale (and, with `zero`, a zero point) for every group of `group` columns, and the values
           that they stand for, which a training step with 4-bit weights goes on with
  linear   a product with weights held that way
  experts  a mixture-of-experts layer for a few tokens: the router's softmax, each token's `k` largest, and the sum of their
           gated feed-forward blocks

`rows` are splats, tokens or output channels, `d` the width (of `pack` the columns, of the products the inputs), `f` the
outputs of `linear` and the hidden width of `experts`. `pad` is the distance between rows beyond their width, in values.
1,000,000 splats with 64 features are the benchmark's scene; the other sizes are generic.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _case(name, op, rows, d, **more):
    c = dict(name=name, op=op, rows=rows, d=d, f=0, dtype="bf16", pad=0, kind="", per_gate=0, gate="", wtype="", train=False,
             group=0, zero=False, experts=0, k=0, act="", residual=False)
    c.update(more)
    return c


def _norm(name, rows, d, kind="rms", per_gate=0, gate="none", wtype="bf16", train=False, **more):
    return _case(name, "norm", rows, d, kind=kind, per_gate=per_gate, gate=gate, wtype=wtype, train=train, **more)


def listed():
    return [
        # one token between two blocks of a wide network: the launch is all there is
        _norm("norm_token", 1, 4096),
        # a training step's tokens, each with a gate of its own
        _norm("norm_train", 8192, 4096, per_gate=1, gate="sigmoid", train=True),
        # the features of the benchmark's scene, every splat a row, with one learned scale a channel for all of them
        _norm("norm_head", 1_000_000, 64, per_gate=1_000_000, wtype="f32", train=True),
        # single precision, ragged: 17 views of 61 tokens that share a gate each
        _norm("norm_odd", 1037, 1000, kind="layer", per_gate=61, dtype="f32", wtype="f32", train=True, pad=24),
        # a wide layer's weights to 4 bits
        _case("pack_wide", "pack", 11264, 4096, group=128),
        # odd columns that end inside a group, master weights in single precision, zero points
        _case("pack_odd", "pack", 5001, 2049, dtype="f32", group=32, zero=True, pad=3),
        # one token through a wide layer in 4 bits: the weights are read once
        _case("q4_token", "linear", 1, 4096, f=11264, group=128),
        # a handful of rows, widths that no tile divides, short groups with zero points
        _case("q4_few", "linear", 7, 2050, f=5001, dtype="f16", group=32, zero=True, pad=6),
        # a prompt through the same layer
        _case("q4_prompt", "linear", 2048, 4096, f=11264, group=128),
        # one token that takes eight of many narrow experts
        _case("experts_token", "experts", 1, 2048, f=1024, experts=64, k=8, act="silu"),
        # a few tokens that take two of sixteen wide experts each: nearly all of them are read
        _case("experts_few", "experts", 16, 2048, f=5632, experts=16, k=2, act="silu", residual=True),
        # more tokens than one tile has, odd widths, half precision
        _case("experts_odd", "experts", 61, 1000, f=1365, experts=10, k=3, dtype="f16", act="gelu", pad=5),
    ]


def draw(rng):
    pick = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    even = lambda v, to, most=1.0: max(to, v // to * to) if rng.random() < most * 0.6 else v  # noqa: E731
    op = rng.choice(["norm", "norm", "pack", "linear", "linear", "experts", "experts"])
    pad = rng.choice([0, 0, 0, 8, 5])
    if op == "norm":
        d = even(pick(3, 8192), 16)
        rows = pick(1, max(2, min(1_000_000, 30_000_000 // d)))
        per_gate = rng.choice([0, 1, rows, pick(1, rows)])
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        c = _norm("", rows, d, kind=rng.choice(["rms", "rms", "layer"]), per_gate=per_gate,
                  gate=rng.choice(["none", "sigmoid"]) if per_gate else "none", dtype=dtype, wtype=rng.choice(["f32", dtype]),
                  train=rng.random() < 0.6, pad=pad)
    elif op == "pack":
        c = _case("", "pack", pick(1, 8192), even(pick(1, 8192), 32), dtype=rng.choice(["f32", "f16", "bf16"]),
                  group=rng.choice([32, 64, 128, 256]), zero=rng.random() < 0.5, pad=pad)
    elif op == "linear":
        c = _case("", "linear", pick(1, rng.choice([16, 256, 2048])), even(pick(33, 8192), 64), f=even(pick(17, 8192), 32),
                  dtype=rng.choice(["f16", "bf16"]), group=rng.choice([32, 64, 128, 256]), zero=rng.random() < 0.5, pad=pad)
    else:
        experts, d = pick(2, 128), even(pick(33, 4096), 32)
        f = even(min(pick(17, 6000), 400_000_000 // (3 * d * experts)), 16)
        c = _case("", "experts", pick(1, 128), d, f=f, experts=experts, k=min(experts, rng.randint(1, 8)),
                  dtype=rng.choice(["f16", "bf16", "bf16"]), act=rng.choice(["silu", "silu", "gelu", "relu"]),
                  residual=rng.random() < 0.5, pad=pad)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------

def _rows(g, rows, cols, dtype, pad=0, scale=1.0):
    """A [rows, cols] matrix of normal values whose rows lie cols + pad apart."""
    x = torch.randn(rows, cols + pad, generator=g, device="cuda", dtype=torch.float32)
    return (x * scale).to(dtype)[:, :cols]


def _ceil(a, b):
    return -(-a // b)


def _scaled(name, g):
    """The gate and its slope."""
    if name == "none":
        return g, torch.ones_like(g)
    s = 1 / (1 + torch.exp(-g))
    return s, s * (1 - s)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, t = case, TYPES[case["dtype"]]
    m, d, f, pad = c["rows"], c["d"], c["f"], c["pad"]
    s = {"case": c}
    if c["op"] == "norm":
        # a block's output of another size than the stream that it joins
        s["x"], s["r"] = _rows(g, m, d, t, pad, 0.5), _rows(g, m, d, t, pad, 2.0)
        s["gate"] = _rows(g, _ceil(m, c["per_gate"]), d, t, pad) if c["per_gate"] else None
        s["w_post"], s["w_pre"] = (1 + _rows(g, 1, d, torch.float32, 0, 0.2)[0]).to(TYPES[c["wtype"]]), (
            1 + _rows(g, 1, d, torch.float32, 0, 0.2)[0]).to(TYPES[c["wtype"]])
        s["scale"] = 0.5
        if c["train"]:
            s["dy"], s["dn"] = _rows(g, m, d, t, pad, 0.1), _rows(g, m, d, t, pad, 0.1)
    elif c["op"] == "pack":
        # a layer's weights: channels of different sizes
        size = torch.exp(torch.rand(m, 1, generator=g, device="cuda") * 2 - 1) * d ** -0.5
        x = torch.randn(m, d + pad, generator=g, device="cuda") * size
        s["x"] = x.to(t)[:, :d]
    elif c["op"] == "linear":
        n = _ceil(d, c["group"])
        s["x"] = _rows(g, m, d, t, pad)
        s["q"] = torch.randint(0, 256, (f, _ceil(d, 2)), generator=g, device="cuda", dtype=torch.uint8)
        s["s"] = ((0.5 + torch.rand(f, n, generator=g, device="cuda")) * (d ** -0.5 / 4.6)).to(t)
        s["z"] = torch.randint(5, 11, (f, n), generator=g, device="cuda", dtype=torch.uint8) if c["zero"] else None
    else:
        e = c["experts"]
        s["x"] = _rows(g, m, d, t, pad)
        s["r"] = _rows(g, m, d, t, pad) if c["residual"] else None
        s["wr"] = _rows(g, e, d, t, 0, d ** -0.5)
        s["wg"], s["wu"] = (_rows(g, e * f, d, t, 0, d ** -0.5) for _ in range(2))
        s["wd"] = _rows(g, e * d, f, t, 0, f ** -0.5)
    if own:
        s["plan"] = _plan(s)
    return s


# ---- one pass --------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _plan(s):
    """The framework's plan of this state's calls, with the buffers it works in: made once, as a program would."""
    from b2ctrain_amd import nn

    c, x = s["case"], s["x"]
    m, d, f = c["rows"], c["d"], c["f"]
    new = lambda *shape, dtype=x.dtype: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    room = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    if c["op"] == "norm":
        out = {"y": new(m, d), "n": new(m, d)}
        p = nn.BlockNorm(x=x, residual=s["r"], y=out["y"], n=out["n"], gate=s["gate"], rows_per_gate=c["per_gate"] or None,
                         gate_act=c["gate"], post=True, w_post=s["w_post"], w_pre=s["w_pre"], kind=c["kind"], eps=EPS, scale=s["scale"])
        if c["train"]:
            out.update(dx=new(m, d), dr=new(m, d), dw_post=torch.empty_like(s["w_post"]), dw_pre=torch.empty_like(s["w_pre"]))
            if s["gate"] is not None:
                out["dgate"] = new(s["gate"].shape[0], d)
            p.gradients(dy=s["dy"], dn=s["dn"], dx=out["dx"], dresidual=out["dr"], dgate=out.get("dgate"), dw_post=out["dw_post"],
                        dw_pre=out["dw_pre"], room=room)
    elif c["op"] == "pack":
        n = _ceil(d, c["group"])
        out = {"values": new(m, d), "s": new(m, n, dtype=torch.bfloat16), "z": new(m, n, dtype=torch.uint8) if c["zero"] else None}
        s["q"] = new(m, _ceil(d, 2), dtype=torch.uint8)
        p = nn.QuantizeGroups(x, s["q"], out["s"], c["group"], zero=out["z"], values=out["values"])
    elif c["op"] == "linear":
        out = {"y": new(m, f)}
        p = nn.Q4Linear(x, s["q"], s["s"], out["y"], c["group"], zero=s["z"], room=room)
    else:
        out = {"y": new(m, d), "index": new(m, c["k"], dtype=torch.int32), "weight": new(m, c["k"], dtype=torch.float32)}
        p = nn.Experts(x, s["wr"], s["wg"], s["wu"], s["wd"], out["y"], c["k"], act=c["act"], normalize=True, residual=s["r"],
                       index=out["index"], weight=out["weight"], room=room)
    return p, out


def _values(q, scale, zero, group, cols):
    """The values that 4 bits stand for."""
    code = torch.stack([q & 15, q >> 4], dim=2).reshape(q.shape[0], -1)[:, :cols].to(scale.dtype)
    wide = lambda v: v.repeat_interleave(group, dim=1)[:, :cols]  # noqa: E731
    return (code - (wide(zero.to(scale.dtype)) if zero is not None else 8)) * wide(scale)


def _run_own(s):
    p, out = s["plan"]
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm":
        p.forward(st)
        if c["train"]:
            p.backward(st)
    else:
        p.run(st)
    return out


def _moments(kind, v):
    """v less its mean, and one over its size."""
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    return v, 1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS)


def _norm_back(kind, unit, size, a):
    """The gradient of v from that of norm(v) = unit."""
    v = a - unit * (a * unit).mean(dim=1, keepdim=True)
    return size * (v - a.mean(dim=1, keepdim=True) if kind == "layer" else v)


def _plain_norm(s):
    c, t, wt = s["case"], s["x"].dtype, s["w_post"].dtype
    m, kind, per = c["rows"], c["kind"], c["per_gate"]
    x, r, w_post, w_pre, scale = s["x"].float(), s["r"].float(), s["w_post"].float(), s["w_pre"].float(), s["scale"]
    if per:
        gate, slope = _scaled(c["gate"], s["gate"].float())
        owner = torch.arange(m, device="cuda") // per
        gate, slope = gate[owner], slope[owner]
    else:
        gate = 1.0
    xc, xs = _moments(kind, x)
    xh = xc * xs
    y = r + scale * gate * (xh * w_post)
    yc, ys = _moments(kind, y)
    yh = yc * ys
    out = {"y": y.to(t), "n": (yh * w_pre).to(t)}
    if c["train"]:
        dn = s["dn"].float()
        full = s["dy"].float() + _norm_back(kind, yh, ys, dn * w_pre)
        dt = scale * gate * full
        out.update(dx=_norm_back(kind, xh, xs, dt * w_post).to(t), dr=full.to(t), dw_post=(dt * xh).sum(dim=0, dtype=torch.float64).to(wt),
                   dw_pre=(dn * yh).sum(dim=0, dtype=torch.float64).to(wt))
        if per:
            each = scale * full * (xh * w_post) * slope
            n = _ceil(m, per)
            if n * per > m:
                each = torch.cat([each, each.new_zeros(n * per - m, c["d"])])
            out["dgate"] = each.reshape(n, per, -1).sum(dim=1, dtype=torch.float64).to(t)
    return out


def _plain_pack(s):
    c, x = s["case"], s["x"].float()
    m, d, g = c["rows"], c["d"], c["group"]
    n = _ceil(d, g)
    if n * g > d:
        x = torch.cat([x, x.new_zeros(m, n * g - d)], dim=1)
    x = x.reshape(m, n, g)
    if c["zero"]:
        lo, hi = x.amin(dim=2).clamp(max=0), x.amax(dim=2).clamp(min=0)
        scale = ((hi - lo) / torch.full_like(hi, 15)).bfloat16()  # by a tensor: by a number it would be a product with 1 / 15
        of = torch.where(scale > 0, scale.float(), 1)
        zero = torch.where(scale > 0, torch.round(-lo / of), 0).clamp(0, 15)
    else:
        top = x.abs().amax(dim=2)
        scale = (top / torch.full_like(top, 7)).bfloat16()
        of = torch.where(scale > 0, scale.float(), 1)
        zero = torch.full_like(of, 8)
    code = torch.where((scale > 0)[:, :, None], torch.round(x / of[:, :, None]), 0) + zero[:, :, None]
    code = code.clamp(0, 15)
    s["q"] = _two_a_byte(code.to(torch.uint8).reshape(m, n * g)[:, :d])
    values = ((code - zero[:, :, None]) * scale.float()[:, :, None]).reshape(m, n * g)[:, :d]
    return {"values": values.to(s["x"].dtype), "s": scale, "z": zero.to(torch.uint8) if c["zero"] else None}


def _two_a_byte(code):
    """The even columns in the low halves of the bytes."""
    if code.shape[1] % 2:
        code = torch.cat([code, code.new_zeros(code.shape[0], 1)], dim=1)
    return code[:, 0::2] | code[:, 1::2] << 4


def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "relu":
        return torch.where(g > 0, g, 0)
    return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))


def _plain_experts(s):
    c, x = s["case"], s["x"].float()
    t, m, d, f, k = s["x"].dtype, c["rows"], c["d"], c["f"], c["k"]
    logits = s["x"].double() @ s["wr"].double().T
    p = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    p = (p / p.sum(dim=1, keepdim=True)).float()
    index = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    weight = torch.gather(p, 1, index)
    weight = weight / weight.sum(dim=1, keepdim=True)
    y = s["r"].float() if s["r"] is not None else torch.zeros(m, d, device="cuda")
    if m * k < c["experts"]:  # the few experts that are chosen
        for i in range(m):
            for j in range(k):
                e = index[i, j:j + 1]
                pick = lambda w, n: w.reshape(c["experts"], n, -1).index_select(0, e)[0].float()  # noqa: E731
                row = x[i:i + 1]
                h = _act(c["act"], row @ pick(s["wg"], f).T) * (row @ pick(s["wu"], f).T)
                y[i] += weight[i, j] * (h @ pick(s["wd"], d).T)[0]
    else:
        for e in range(c["experts"]):
            of = torch.where(index == e, weight, 0).sum(dim=1, keepdim=True)
            wg, wu, wd = s["wg"][e * f:(e + 1) * f], s["wu"][e * f:(e + 1) * f], s["wd"][e * d:(e + 1) * d]
            h = _act(c["act"], x @ wg.float().T) * (x @ wu.float().T)
            y = y + of * (h @ wd.float().T)
    return {"y": y.to(t), "index": index.int(), "weight": weight}


def _run_plain(s):
    c = s["case"]
    if c["op"] == "norm":
        return _plain_norm(s)
    if c["op"] == "pack":
        return _plain_pack(s)
    if c["op"] == "linear":
        w = _values(s["q"], s["s"].float(), s["z"], c["group"], c["d"])
        return {"y": (s["x"].float() @ w.T).to(s["x"].dtype)}
    return _plain_experts(s)


# ---- what it has to cost, and what it should be ----------------------------------------------------------

def work(case):
    c = case
    m, d, f = c["rows"], c["d"], c["f"]
    b = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        gates, w = _ceil(m, c["per_gate"]) * d if c["per_gate"] else 0, 2 * d * (4 if c["wtype"] == "f32" else 2)
        bytes_, flops = b * (4 * m * d + gates) + w, 12 * m * d
        if c["train"]:
            bytes_, flops = bytes_ + b * (4 * m * d + gates) + w, flops + 24 * m * d
        return {"bytes": bytes_, "flops": flops}
    if c["op"] == "pack":
        return {"bytes": m * (2 * d * b + _ceil(d, 2) + _ceil(d, c["group"]) * (2 + c["zero"])), "flops": 4 * m * d}
    if c["op"] == "linear":
        return {"bytes": b * m * (d + f) + f * (_ceil(d, 2) + _ceil(d, c["group"]) * (2 + c["zero"])), "flops": 2 * m * d * f}
    e, k = c["experts"], c["k"]
    chosen = min(e, m * k) if m == 1 else e * (1 - (1 - k / e) ** m)  # the experts that tokens meet, if each takes any k
    return {"bytes": int(b * (m * d * (2 + c["residual"]) + e * d + chosen * 3 * d * f)), "flops": m * (2 * e * d + 6 * k * d * f)}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"norm": _exact_norm, "pack": _exact_pack, "linear": _exact_linear, "experts": _exact_experts}[c["op"]](c, s)


def _exact_norm(c, s):
    m, d, per = c["rows"], c["d"], c["per_gate"]
    x, r, wa, wb = (s[k].double() for k in ("x", "r", "w_post", "w_pre"))
    centre = c["kind"] == "layer"

    def unit(v):
        if centre:
            v = v - v.sum(1, keepdim=True) / d
        size = torch.rsqrt(v.pow(2).sum(1, keepdim=True) / d + EPS)
        return v * size, size

    def back(u, size, a):
        # the gradient less what of it points along the unit row (and along ones)
        along = u * ((a * u).sum(1, keepdim=True) / d)
        if centre:
            along = along + a.sum(1, keepdim=True) / d
        return (a - along) * size

    if per:
        raw = s["gate"].double().repeat_interleave(per, 0)[:m]
        g = raw if c["gate"] == "none" else torch.sigmoid(raw)
    else:
        g = torch.ones((), dtype=torch.float64, device=x.device)
    u, su = unit(x)
    y = torch.addcmul(r, g, u * wa, value=s["scale"])
    v, sv = unit(y)
    out = {"y": y, "n": v * wb}
    if c["train"]:
        dn = s["dn"].double()
        dy = s["dy"].double() + back(v, sv, dn * wb)
        dt = s["scale"] * g * dy
        out.update(dx=back(u, su, dt * wa), dr=dy, dw_post=torch.linalg.vecdot(dt, u, dim=0), dw_pre=torch.linalg.vecdot(dn, v, dim=0))
        if per:
            dg = s["scale"] * dy * u * wa * (1 if c["gate"] == "none" else g * (1 - g))
            to = torch.arange(m, device=x.device) // per
            out["dgate"] = torch.zeros(_ceil(m, per), d, dtype=torch.float64, device=x.device).index_add_(0, to, dg)
    return out


def _exact_pack(c, s):
    """The scale is formed in single precision and rounded to bfloat16, and the quotient is one of single precision: of numbers of 24 bits,
    it is the one in 64 bits, rounded."""
    m, d, g = c["rows"], c["d"], c["group"]
    n = _ceil(d, g)
    x = torch.zeros(m, n * g, dtype=torch.float64, device="cuda")
    x[:, :d] = s["x"].double()
    x = x.view(m, n, g)
    top, low = x.max(2).values, x.min(2).values
    if c["zero"]:
        low = torch.minimum(low, torch.zeros_like(low))
        reach = (torch.maximum(top, torch.zeros_like(top)) - low).float().double() / torch.full_like(top, 15)
    else:
        reach = torch.maximum(top, -low) / torch.full_like(top, 7)
    step = reach.float().to(torch.bfloat16)
    wide = step.double()
    there = wide > 0
    zero = torch.where(there, -low / wide, 0.0).float().round().double() if c["zero"] else torch.full_like(wide, 8.0)
    code = torch.where(there[:, :, None], x / wide[:, :, None], 0.0).float().round().double() + zero[:, :, None]
    values = (code.clamp(0, 15) - zero[:, :, None]) * wide[:, :, None]
    return {"values": values.view(m, n * g)[:, :d], "s": step, "z": zero.to(torch.uint8) if c["zero"] else None}


def _exact_linear(c, s):
    m, d, f, g = c["rows"], c["d"], c["f"], c["group"]
    x, y = s["x"].double(), torch.zeros(m, f, dtype=torch.float64, device="cuda")
    for i in range(0, d, g):  # group by group
        q = s["q"][:, i // 2:_ceil(min(i + g, d), 2)]
        code = torch.empty(f, 2 * q.shape[1], dtype=torch.float64, device="cuda")
        code[:, 0::2], code[:, 1::2] = (q % 16).double(), (q // 16).double()
        code = code[:, :min(g, d - i)] - (s["z"][:, i // g].double()[:, None] if c["zero"] else 8.0)
        y += torch.mm(x[:, i:i + g], code.t()) * s["s"][:, i // g].double()
    return {"y": y}


def _exact_experts(c, s):
    m, d, f, e, k = c["rows"], c["d"], c["f"], c["experts"], c["k"]
    x = s["x"].double()
    logits = torch.mm(x, s["wr"].double().t())
    order = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    share = torch.softmax(torch.take_along_dim(logits, order, 1), dim=1)  # of the chosen alone: what renormalising gives
    y = s["r"].double() if c["residual"] else torch.zeros(m, d, dtype=torch.float64, device="cuda")
    for i in range(e):
        at, slot = (order == i).nonzero(as_tuple=True)
        if at.numel() == 0:
            continue
        wg, wu, wd = (s[n].view(e, -1, s[n].shape[1])[i].double() for n in ("wg", "wu", "wd"))
        g, u = torch.mm(x[at], wg.t()), torch.mm(x[at], wu.t())
        a = g * torch.sigmoid(g) if c["act"] == "silu" else g.clamp(min=0) if c["act"] == "relu" else g * torch.special.ndtr(g)
        y.index_add_(0, at, torch.mm(a * u, wd.t()) * share[at, slot][:, None])
    return {"y": y, "index": order.int(), "weight": share}
