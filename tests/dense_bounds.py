"""How far the block's gradients may be off, term by term as they are formed: g, u, act(g) and u act'(g) stay in single precision,
h, dg and du are rounded once, for the products that take them."""
import numpy as np

from b2ctrain_amd import nn
from tests import dense_util as U


def grads_bound(x, wg, wu, wd, name, dtype, dy, m):
    """(the gradients in 64 bits, how far each value may be from them)."""
    e, b = U.UNIT[dtype], lambda n: (n + 8) * U.F32_SUM
    tiny = 2.0 ** -25 if dtype == nn.F16 else 2.0 ** -134  # half the distance of the type's subnormals
    rows, di = x.shape
    f, do = wg.shape[0], wd.shape[0]
    g, u = x @ wg.T, x @ wu.T
    a, d = U.act(name, g)
    dz = dy * m
    dh = dz @ wd
    eg, eu, edh = b(di) * (abs(x) @ abs(wg).T), b(di) * (abs(x) @ abs(wu).T), b(do) * (abs(dz) @ abs(wd))
    ea, ed = U.SLOPE[name] * eg + U.ACT_EPS * (abs(a) + 1), U.CURVE[name] * eg + U.ACT_EPS * 4
    if name == "relu":  # a g within its error of zero may take either slope
        ed = ed + (abs(g) <= eg)
    eh = ea * (abs(u) + eu) + abs(a) * eu + e * abs(a * u) + tiny
    edg = (abs(dh) + edh) * ((abs(u) + eu) * ed + eu * abs(d)) + edh * abs(u * d) + e * abs(dh * u * d) + tiny
    edu = (abs(dh) + edh) * ea + edh * abs(a) + e * abs(dh * a) + tiny
    dg, du, h = dh * u * d, dh * a, a * u
    ref = U.block_grads(x, wg, wu, wd, name, dy, m)
    off = {"dx": edg @ abs(wg) + edu @ abs(wu) + b(2 * f) * (abs(dg) @ abs(wg) + abs(du) @ abs(wu)),
           "dw_gate": edg.T @ abs(x) + b(rows) * (abs(dg).T @ abs(x)), "dw_up": edu.T @ abs(x) + b(rows) * (abs(du).T @ abs(x)),
           "dw_down": abs(dz).T @ eh + b(rows) * (abs(dz).T @ abs(h))}
    # second order: at most 2 e of what is of the first, and the output's own rounding
    return ref, {k: off[k] * (1 + 4 * e) + e * (abs(ref[k]) + off[k]) + tiny for k in off}


def rounded_grads(x, wg, wu, wd, name, dtype, dy, m, factors=False, inputs=False):
    """The gradients with those roundings and 64 bits elsewhere; `factors`: act(g) and u act'(g) are rounded too, as they would be if they
    were kept in 16 bits; `inputs`: g and u, likewise."""
    r = lambda v: U.rounded(v, dtype)  # noqa: E731
    g, u = x @ wg.T, x @ wu.T
    a0, _ = U.act(name, g)
    h = r(a0 * u)
    if inputs:
        g, u = r(g), r(u)
        a0, _ = U.act(name, g)
        h = r(a0 * u)
    a, d = U.act(name, g)
    fa, fb = (r(a), r(u * d)) if factors else (a, u * d)
    dz = dy * m
    dh = dz @ wd
    dg, du = r(dh * fb), r(dh * fa)
    return {k: r(v) for k, v in {"dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dz.T @ h}.items()}


# Sizes at which an output is one term or two, so that its rounding shows: rows, d_in, d_hidden, d_out.
SINGLE = [(1, 16, 40, 24), (1, 200, 70, 136), (50, 24, 1, 16), (50, 136, 1, 200), (300, 144, 1, 40), (1, 1, 1, 1)]


def make(rows, di, f, do, dtype, seed):
    g = np.random.default_rng(seed)
    q = lambda *s, k=1.0: U.rounded(g.standard_normal(s) * k, dtype)  # noqa: E731
    return q(rows, di), q(f, di, k=di ** -0.5), q(f, di, k=di ** -0.5), q(do, f, k=f ** -0.5), q(rows, do, k=0.3)
