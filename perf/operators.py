"""The dense operators of a learned head over splats or image tokens, as cases to be timed and compared.

  op       one pass
  ffn      the gated feed-forward block y = r + dropout((act(x Wg') * (x Wu')) Wd'); with `train` also its backward
           pass: the gradients of x and of the three weights
  dropout  y = r + dropout(x) from a counter-based generator, and the gradient of x
  linear   a product in 8-bit integers: x quantised by rows, weights held quantised by channels
  block    the feed-forward block in 8-bit integers, as a renderer runs a trained head

`rows` are splats or tokens, `d` the input and output width, `f` the hidden width (for `linear`: `d` inputs, `f`
outputs). `pad` is the distance between rows beyond their width, in values. The widths of the small heads go with
1,000,000 splats, the benchmark's scene; the others are generic.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ffn(name, rows, d, f, dtype="bf16", act="silu", train=False, p=0.0, residual=False, pad=0):
    return dict(name=name, op="ffn", rows=rows, d=d, f=f, dtype=dtype, act=act, train=train, p=p, residual=residual, pad=pad)


def _drop(name, rows, cols, dtype="bf16", p=0.1, residual=True, pad=0):
    return dict(name=name, op="dropout", rows=rows, d=cols, f=0, dtype=dtype, act="", train=True, p=p, residual=residual, pad=pad)


def _i8(name, op, rows, d, f, dtype="bf16", act="silu", pad=0):
    return dict(name=name, op=op, rows=rows, d=d, f=f, dtype=dtype, act=act if op == "block" else "", train=False, p=0.0, residual=False, pad=pad)


def listed():
    return [
        # a handful of rows through a small head: the launches are all there is
        _ffn("ffn_tiny", 7, 96, 256, dtype="f16", act="gelu"),
        # one token answered by a wide block: the weights are read once
        _ffn("ffn_token", 1, 4096, 11264),
        # a prompt, or a frame of tokens, through the same block
        _ffn("ffn_prompt", 4096, 4096, 11264),
        # a training step of an ordinary block, with dropout and the residual sum
        _ffn("ffn_train", 8192, 2048, 5632, train=True, p=0.1, residual=True),
        # widths and rows that no tile divides, half precision
        _ffn("ffn_train_odd", 1037, 1000, 2730, dtype="f16", act="gelu", train=True, pad=24),
        # the appearance head of the benchmark's scene: every splat a row
        _ffn("ffn_head", 1_000_000, 64, 256, train=True, p=0.1),
        # dropout of a block's output in training, added to the residual stream
        _drop("drop_train", 8192, 4096),
        # dropout over the splats' colour coefficients, single precision, an odd count and a padded layout
        _drop("drop_lanes", 333_333, 45, dtype="f32", p=0.25, residual=False, pad=3),
        # one token through a layer held in 8 bits
        _i8("linear_token", "linear", 1, 4096, 4096),
        # a ragged batch through one
        _i8("linear_odd", "linear", 1333, 2050, 5001, dtype="f16"),
        # the trained appearance head in 8 bits over the whole scene, as a frame is rendered
        _i8("block_head", "block", 1_000_000, 64, 256),
        # a wide block in 8 bits over a prompt
        _i8("block_prompt", "block", 4096, 4096, 11264),
    ]


def draw(rng):
    pick = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["ffn", "ffn", "ffn", "dropout", "linear", "block"])
    if op == "dropout":
        cols = pick(3, 8192)
        c = _drop("", pick(1, max(1, 30_000_000 // cols)), cols, dtype=rng.choice(["f32", "f16", "bf16"]),
                  p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9]), residual=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 8, 24]))
    else:
        # heads over splats, blocks over tokens, or a few tokens at a time
        kind = rng.choice(["head", "block", "block", "token"])
        if kind == "head":
            rows, d, f = pick(1000, 700_000), pick(16, 128), pick(32, 384)
        elif kind == "block":
            rows, d, f = pick(64, 6000), pick(256, 2800), pick(256, 7000)
        else:
            rows, d, f = pick(1, 48), pick(64, 4096), pick(128, 11264)
        if rng.random() < 0.6:  # widths are mostly multiples of a tile's side, but not always
            d, f = max(16, d // 16 * 16), max(32, f // 32 * 32)
        dtype = rng.choice(["f16", "bf16", "bf16"])
        pad = rng.choice([0, 0, 0, 8, 5])
        if op == "ffn":
            train = kind != "token" and rng.random() < 0.6
            c = _ffn("", rows, d, f, dtype=dtype, act=rng.choice(["silu", "silu", "gelu", "relu"]), train=train,
                     p=rng.choice([0.0, 0.1, 0.3]) if train else 0.0, residual=rng.random() < 0.5, pad=pad)
        else:
            c = _i8("", op, rows, d, f, dtype=dtype, act=rng.choice(["silu", "gelu", "relu"]), pad=pad)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------

def _rows(g, rows, cols, dtype, pad, scale=1.0):
    """A [rows, cols] matrix of normal values whose rows lie cols + pad apart."""
    x = torch.randn(rows, cols + pad, generator=g, device="cuda", dtype=torch.float32)
    return (x * scale).to(dtype)[:, :cols]


def _quantised(w):
    """(values in 8 bits, a scale for each row): the weights of a trained layer, laid out once."""
    s = w.abs().amax(dim=1) / 127
    return torch.round(w / s[:, None]).clamp(-127, 127).to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, t = case, TYPES[case["dtype"]]
    m, d, f, pad = c["rows"], c["d"], c["f"], c["pad"]
    s = {"case": c, "seed": seed * 0x9E3779B97F4A7C15 % (1 << 63), "stream": 1000 + seed % 1000}
    s["x"] = _rows(g, m, d, t, pad)
    s["r"] = _rows(g, m, d, t, pad) if c["residual"] else None
    if c["train"]:
        s["dy"] = _rows(g, m, d, t, pad, 0.1)
    if c["op"] == "ffn":
        s["wg"], s["wu"] = (_rows(g, f, d, t, 0, d ** -0.5) for _ in range(2))
        s["wd"] = _rows(g, d, f, t, 0, f ** -0.5)
    elif c["op"] == "linear":
        s["w"], s["sw"] = _quantised(_rows(g, f, d, torch.float32, 0, d ** -0.5))
    elif c["op"] == "block":
        s["wg"], s["sg"] = _quantised(_rows(g, f, d, torch.float32, 0, d ** -0.5))
        s["wu"], s["su"] = _quantised(_rows(g, f, d, torch.float32, 0, d ** -0.5))
        s["wd"], s["sd"] = _quantised(_rows(g, d, f, torch.float32, 0, f ** -0.5))
    return s


# ---- one pass --------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _plan(s):
    """The framework's plan of this state's calls, with the buffers it works in: made once, as a program would."""
    if "plan" in s:
        return s["plan"]
    from b2ctrain_amd import nn

    c, x = s["case"], s["x"]
    m, d, f = c["rows"], c["d"], c["f"]
    new = lambda *shape: torch.empty(*shape, dtype=x.dtype, device="cuda")  # noqa: E731
    room = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    out = {"y": new(m, f if c["op"] == "linear" else d)}
    if c["op"] == "dropout":
        out["dx"] = new(m, d)
        p = (nn.Dropout(x, out["y"], c["p"], s["seed"], s["stream"], residual=s["r"]),
             nn.Dropout(s["dy"], out["dx"], c["p"], s["seed"], s["stream"]))
    elif c["op"] == "linear":
        p = nn.I8Linear(x, s["w"], s["sw"], out["y"], room=room)
    elif c["op"] == "block":
        p = nn.I8FeedForward(x, s["wg"], s["sg"], s["wu"], s["su"], s["wd"], s["sd"], out["y"], act=c["act"], room=room)
    else:
        p = nn.FeedForward(x, s["wg"], s["wu"], s["wd"], out["y"], act=c["act"], residual=s["r"], p=c["p"], seed=s["seed"],
                           stream_id=s["stream"], train=c["train"], room=room)
        if c["train"]:
            out.update(dx=new(m, d), dwg=new(f, d), dwu=new(f, d), dwd=new(d, f))
            p.gradients(s["dy"], dx=out["dx"], dw_gate=out["dwg"], dw_up=out["dwu"], dw_down=out["dwd"], room=room)
    s["plan"] = (p, out)
    return s["plan"]


def _run_own(s):
    p, out = _plan(s)
    c, st = s["case"], _stream()
    if c["op"] == "dropout":
        p[0].run(st)
        p[1].run(st)
    elif c["op"] == "ffn":
        p.forward(st)
        if c["train"]:
            p.backward(st)
    else:
        p.run(st)
    return out


def _keep(rows, cols, p, seed, stream):
    """Which values dropout keeps: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) under the key `seed` at the counters
    (value's index / 8, stream), sixteen bits for each value, low halves first; kept from round(65536 p) up."""
    n, low = rows * cols, 0xFFFFFFFF
    at = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)
    full = torch.full_like(at, stream & low)
    c = [at & low, at >> 32, full, torch.full_like(at, stream >> 32)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32 & low) ^ c[1] ^ k0, b & low, (a >> 32 & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    bits = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1).reshape(-1)[:n]
    return (bits >= _threshold(p)).reshape(rows, cols)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _scale(p):
    return 65536 / (65536 - _threshold(p))


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "relu":
        return torch.where(g > 0, g, 0), (g > 0).to(g.dtype)
    phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _by_rows(x):
    s = x.abs().amax(dim=1) / 127
    return torch.where(s[:, None] > 0, torch.round(x / s[:, None]), 0), s


def _run_plain(s):
    c, x = s["case"], s["x"].float()
    t = s["x"].dtype
    if c["op"] == "linear":
        q, sx = _by_rows(x)
        return {"y": ((q @ s["w"].float().T) * sx[:, None] * s["sw"]).to(t)}
    if c["op"] == "block":
        q, sx = _by_rows(x)
        h = _act(c["act"], (q @ s["wg"].float().T) * sx[:, None] * s["sg"])[0] * ((q @ s["wu"].float().T) * sx[:, None] * s["su"])
        q, sh = _by_rows(h)
        return {"y": ((q @ s["wd"].float().T) * sh[:, None] * s["sd"]).to(t)}
    drop = lambda v: v  # noqa: E731
    if c["p"] > 0:
        keep, scale = _keep(c["rows"], c["d"], c["p"], s["seed"], s["stream"]), _scale(c["p"])
        drop = lambda v: torch.where(keep, v * scale, 0)  # noqa: E731
    add = (lambda v: v + s["r"].float()) if s["r"] is not None else (lambda v: v)
    if c["op"] == "dropout":
        return {"y": add(drop(x)).to(t), "dx": drop(s["dy"].float()).to(t)}
    wg, wu, wd = s["wg"].float(), s["wu"].float(), s["wd"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(c["act"], g)
    h = a * u
    out = {"y": add(drop(h @ wd.T)).to(t)}
    if c["train"]:
        dz = drop(s["dy"].float())
        dh = dz @ wd
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).to(t), dwg=(dg.T @ x).to(t), dwu=(du.T @ x).to(t), dwd=(dz.T @ h).to(t))
    return out


# ---- what it has to cost, and what it should be ----------------------------------------------------------

def work(case):
    c = case
    m, d, f = c["rows"], c["d"], c["f"]
    b = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "dropout":
        return {"bytes": b * m * d * (4 + c["residual"]), "flops": 4 * m * d}
    if c["op"] == "linear":
        return {"bytes": b * m * (d + f) + f * (d + 4), "flops": 2 * m * d * f}
    if c["op"] == "block":
        return {"bytes": b * 2 * m * d + 3 * d * f + 4 * (2 * f + d), "flops": 6 * m * d * f}
    bytes_, flops = b * (m * d * (2 + c["residual"]) + 3 * d * f), 6 * m * d * f
    if c["train"]:
        bytes_, flops = bytes_ + b * (2 * m * d + 3 * d * f), 3 * flops
    return {"bytes": bytes_, "flops": flops}


def _keep_exact(rows, cols, p, seed, stream):
    """The same choice on the host, in numpy's unsigned integers."""
    n = rows * cols
    at = np.arange(-(-n // 8), dtype=np.uint64)
    w = np.empty((at.size, 4), np.uint32)
    w[:, 0], w[:, 1] = at.astype(np.uint32), (at >> np.uint64(32)).astype(np.uint32)
    w[:, 2], w[:, 3] = np.uint32(stream & 0xFFFFFFFF), np.uint32(stream >> 32)
    key = [seed % (1 << 32), seed // (1 << 32)]
    for r in range(10):
        p0 = w[:, 0].astype(np.uint64) * np.uint64(0xD2511F53)
        p1 = w[:, 2].astype(np.uint64) * np.uint64(0xCD9E8D57)
        k0, k1 = (np.uint32((key[i] + r * step) % (1 << 32)) for i, step in ((0, 0x9E3779B9), (1, 0xBB67AE85)))
        w = np.stack([(p1 >> np.uint64(32)).astype(np.uint32) ^ w[:, 1] ^ k0, p1.astype(np.uint32),
                      (p0 >> np.uint64(32)).astype(np.uint32) ^ w[:, 3] ^ k1, p0.astype(np.uint32)], axis=1)
    bits = w.reshape(-1).view(np.uint16)[:n]  # little-endian: the low half of a word comes first
    return torch.from_numpy((bits >= round(p * 65536)).reshape(rows, cols)).cuda()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    x = s["x"].double()
    if c["op"] in ("linear", "block"):
        def dense(v, w, sw):
            scale = v.abs().max(dim=1, keepdim=True).values / 127
            q = torch.nan_to_num(v / scale).round()
            return torch.mm(q, w.double().t()) * scale * sw.double()

        if c["op"] == "linear":
            return {"y": dense(x, s["w"], s["sw"])}
        g, u = dense(x, s["wg"], s["sg"]), dense(x, s["wu"], s["su"])
        return {"y": dense(_gate_exact(c["act"], g)[0] * u, s["wd"], s["sd"])}
    factor = 1.0
    if c["p"] > 0:
        kept = _keep_exact(c["rows"], c["d"], c["p"], s["seed"], s["stream"])
        factor = kept.double() / (1 - round(c["p"] * 65536) / 65536)
    r = s["r"].double() if c["residual"] else 0.0
    if c["op"] == "dropout":
        return {"y": x * factor + r, "dx": s["dy"].double() * factor}
    wg, wu, wd = (s[k].double() for k in ("wg", "wu", "wd"))
    g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    a, slope = _gate_exact(c["act"], g)
    out = {"y": torch.mm(a * u, wd.t()) * factor + r}
    if c["train"]:
        dz = s["dy"].double() * factor
        dh = torch.mm(dz, wd)
        out["dwd"] = torch.mm(dz.t(), a * u)
        dg, du = dh * u * slope, dh * a
        out["dx"] = torch.mm(dg, wg) + torch.mm(du, wu)
        out["dwg"], out["dwu"] = torch.mm(dg.t(), x), torch.mm(du.t(), x)
    return out


def _gate_exact(name, g):
    if name == "relu":
        return g.clamp(min=0), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    phi = torch.special.ndtr(g)
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
