"""The norms between blocks, 4-bit weights and experts restated in 64 bits, each with how far a kernel that sums in single precision and
rounds where the documentation says may be off, value by value."""
import numpy as np

from b2ctrain_amd import nn
from tests import dense_util as U

R = 2.0 ** -24  # a rounding in single precision
SUM = 64 * R    # a row's sum, relative to its terms' magnitudes: a thread adds up to 32, then six steps in a wave and sixteen waves
TINY = {nn.F32: 2.0 ** -149, nn.F16: 2.0 ** -25, nn.BF16: 2.0 ** -133}


def mean(v):
    return v.mean(axis=1, keepdims=True)


class Norm:
    """norm(v) as `u`, off by at most `eu`; one over its size as `size`, off by `es` of itself. `ev`: how far v may be off."""

    def __init__(self, v, ev, kind, eps):
        self.kind = kind
        c, ec = v, ev
        if kind == "layer":
            c = v - mean(v)
            ec = ev + mean(ev) + SUM * mean(abs(v)) + R * abs(c)
        self.size = 1 / np.sqrt(mean(c * c) + eps)
        self.u = c * self.size
        # the sum of squares moves by at most 2 rms(c) rms(ec), its root by rms(ec)
        self.es = (np.sqrt(mean(ec * ec)) * self.size + SUM / 2 + 4 * R) * 1.01
        self.eu = self.size * ec * 1.01 + abs(self.u) * (self.es + R)

    def back(self, a, ea):
        """The gradient of v from a, that of u; and how far it may be off."""
        u, eu = self.u, self.eu
        m = mean(a) if self.kind == "layer" else 0 * mean(a)
        em = (mean(ea) + SUM * mean(abs(a))) if self.kind == "layer" else 0 * m
        along = mean(a * u)
        ealong = mean(ea * abs(u) + abs(a) * eu) + SUM * mean(abs(a * u))
        inner = a - m - u * along
        e = ea + em + abs(u) * ealong + eu * abs(along) + 4 * R * (abs(a) + abs(m) + abs(u * along))
        return self.size * inner, self.size * (e + abs(inner) * (self.es + 2 * R)) * 1.01


def block_norm(dtype, w_dtype, x=None, r=None, gate=None, per=1, act="none", post=False, w_post=None, w_pre=None, kind="rms", eps=1e-6,
               scale=1.0, want_n=True, dy=None, dn=None, grad_dtype=None):
    """{name: (value, how far it may be off)}."""
    e, out = U.UNIT[dtype], {}
    scale, eps = float(np.float32(scale)), float(np.float32(eps))
    some = x if x is not None else r
    rows, d = some.shape
    zero = np.zeros((rows, d))
    held = lambda v, ev, t=dtype: (v, ev + U.UNIT[t] * (abs(v) + ev) + TINY[t])  # noqa: E731
    wa, wb = (np.ones(d) if w is None else w for w in (w_post, w_pre))
    if x is not None:
        if gate is None:
            g, eg, slope, eslope = np.ones((rows, d)), zero, np.ones((rows, d)), zero
        else:
            raw = gate[np.arange(rows) // per]
            g, eg, slope, eslope = raw, zero, np.ones((rows, d)), zero
            if act == "sigmoid":  # the exponential's argument is rounded, then itself, the sum and its reciprocal
                g = 1 / (1 + np.exp(-raw))
                eg = g * (abs(raw) + 8) * 2 * R
                slope, eslope = g * (1 - g), 2 * eg + 2 * R
        if post:
            px = Norm(x, zero, kind, eps)
            u, eu = px.u, px.eu
            t, et = u * wa, eu * abs(wa) + R * abs(u * wa)
        else:
            u, eu, t, et = x, zero, x, zero
        y = scale * g * t + (0 if r is None else r)
        ey = abs(scale) * (abs(g) * et + abs(t) * eg) + 4 * R * abs(scale * g * t) + R * abs(y)
        out["y"] = held(y, ey)
    else:
        y, ey = r, zero
    py = Norm(y, ey, kind, eps) if want_n or dn is not None else None
    if want_n:
        out["n"] = held(py.u * wb, py.eu * abs(wb) + R * abs(py.u * wb))
    if dy is None and dn is None:
        return out
    gt = w_dtype if grad_dtype is None else grad_dtype
    full, ef = (zero, zero) if dy is None else (dy, zero)
    if dn is not None:
        b, eb = py.back(dn * wb, R * abs(dn * wb))
        full, ef = full + b, eb + R * abs(full + b)
        terms = dn * py.u
        out["dw_pre"] = held(terms.sum(0), (abs(dn) * py.eu).sum(0) + (rows + 16) * R * abs(terms).sum(0), gt)
    out["dresidual"] = held(full, ef)
    if x is None:
        return out
    dg = scale * full * t * slope
    edg = abs(scale) * (abs(t * slope) * ef + abs(full * slope) * et + abs(full * t) * eslope) + 5 * R * abs(dg)
    if gate is not None:
        starts = np.arange(0, rows, per)
        value, off, size = (np.add.reduceat(v, starts, axis=0) for v in (dg, edg, abs(dg)))
        out["dgate"] = held(value, off + (min(per, rows) + 16) * R * size * (per > 1))
    dt, edt = scale * g * full, abs(scale) * (abs(g) * ef + abs(full) * eg) + 3 * R * abs(scale * g * full)
    if post:
        terms = dt * u
        out["dw_post"] = held(terms.sum(0), (edt * abs(u) + abs(dt) * eu).sum(0) + (rows + 16) * R * abs(terms).sum(0), gt)
        dt, edt = px.back(dt * wa, edt * abs(wa) + R * abs(dt * wa))
    out["dx"] = held(dt, edt)
    return out


# ---- 4 bits ------------------------------------------------------------------------------------------------

def groups(cols, group):
    return -(-cols // group)


def quantised4(x, group, zeros, scale_dtype):
    """(codes, scales as stored, zero points, values in single precision) of x, in single precision as the documentation has it."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    n = groups(cols, group)
    v = np.zeros((rows, n * group), np.float32)
    v[:, :cols] = x
    v = v.reshape(rows, n, group)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(v).all(axis=2)
        lo, hi = np.minimum(np.nan_to_num(v, nan=0).min(axis=2), 0), np.maximum(np.nan_to_num(v, nan=0).max(axis=2), 0)
        reach = (hi - lo) / np.float32(15) if zeros else np.maximum(hi, -lo) / np.float32(7)
        stored = U.store(np.where(bad, np.float32(np.nan), reach), scale_dtype)
        s = U.value(stored, scale_dtype).astype(np.float32)
        fine = (s > 0) & np.isfinite(s)
        safe = np.where(fine, s, np.float32(1))
        z = np.where(fine, np.clip(np.rint(-lo / safe), 0, 15), 0) if zeros else np.full(s.shape, 8.0)
        code = np.where(fine[:, :, None], np.clip(np.rint(v / safe[:, :, None]) + z[:, :, None], 0, 15), z[:, :, None])
        values = ((code - z[:, :, None]).astype(np.float32) * s[:, :, None]).reshape(rows, -1)[:, :cols]
    return code.reshape(rows, -1)[:, :cols].astype(np.uint8), stored, z.astype(np.uint8), values


def packed(code):
    """Two columns a byte."""
    rows, cols = code.shape
    c = np.zeros((rows, cols + cols % 2), np.uint8)
    c[:, :cols] = code
    return c[:, 0::2] | c[:, 1::2] << 4


def q4_linear(x, code, scale, zero, group, dtype, few):
    """y and how far it may be off: of a few rows a group's sums hold (BASE + code) x, else w is rounded once."""
    k = x.shape[1]
    wide = lambda v: np.repeat(v, group, axis=1)[:, :k].astype(np.float64)  # noqa: E731
    s = wide(scale)
    w = (code.astype(np.float64) - wide(zero)) * s
    y = x @ w.T
    if few:
        base = 128 if dtype == nn.BF16 else 64
        off = (2 * (group + 8) * R) * (abs(x) @ ((base + 16) * abs(s)).T) + (k / group + 16) * R * (abs(x) @ abs(w).T)
    else:
        off = (U.UNIT[dtype] * abs(x)) @ abs(w).T * 1.01 + (k + 8) * R * (abs(x) @ abs(w).T) + TINY[dtype] * abs(x).sum(1, keepdims=True)
    return y, off + U.UNIT[dtype] * (abs(y) + off) + TINY[dtype]


# ---- experts -----------------------------------------------------------------------------------------------

def route(x, wr, k, normalize):
    logits = x @ wr.T
    index = np.argsort(-logits, axis=1, kind="stable")[:, :k]
    p = np.exp(logits - logits.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    share = np.take_along_axis(p, index, 1)
    return index, share / share.sum(axis=1, keepdims=True) if normalize else share


SHARE = 2.0 ** -20  # exponentials of differences rounded to single precision, a sum of up to 64 (or a tree of 1024), a quotient


def experts(x, wr, wg, wu, wd, k, name, dtype, normalize=True, r=None):
    """(index, share, y, how far y may be off)."""
    e = len(wr)
    f, o = len(wg) // e, len(wd) // e
    index, share = route(x, wr, k, normalize)
    y, off = np.zeros((len(x), o)), np.zeros((len(x), o))
    for i in range(e):
        at, slot = np.nonzero(index == i)
        if not len(at):
            continue
        w = wg[i * f:(i + 1) * f], wu[i * f:(i + 1) * f], wd[i * o:(i + 1) * o]
        p = share[at, slot][:, None]
        v = U.block(x[at], *w, name)
        y[at] += p * v
        off[at] += p * (U.block_bound(x[at], *w, name, dtype) - U.UNIT[dtype] * abs(v) + (SHARE + (k + 2) * R) * abs(v))
    if r is not None:
        y = y + r
    return index, share, y, off + R * abs(y) + U.UNIT[dtype] * (abs(y) + off) + TINY[dtype]
