"""How far outputs are off on the whole, against how far their own rounding leaves them: what bounds that hold for every single value
cannot see."""
import numpy as np

from tests import dense_util as U
from tests import more_util as V


def rms(v):
    return float(np.sqrt(np.mean(np.square(v, dtype=np.float64))))


def excess(got, want, dtype):
    """The root mean square error of `got`, in units of that of `want` rounded once to `dtype`."""
    return rms(got - want) / rms(U.rounded(want, dtype) - want)


# What else a kernel does may add up to a third of the output's own rounding, in squares: 1.05. Sums of up to 5000 products in single precision add
# about sqrt(5000) 2^-24 of the terms' size to a y of sqrt(5000) times it, some 2^-22 with the base of the codes, against 2^-9.2 or 2^-12.2 for y's
# rounding; two thousand outputs tell the mean of their squares to within 3%.
MOST = 1.05


def weights4(rows, k, n, group, zeros, dtype):
    """x, codes, scales, zero points and the weights that they stand for."""
    g = np.random.default_rng(rows + k + n + group)
    x = U.rounded(g.standard_normal((rows, k)), dtype)
    code, m = g.integers(0, 16, (n, k)).astype(np.uint8), V.groups(k, group)
    scale = U.rounded((0.5 + g.random((n, m))) / (4.6 * np.sqrt(k)), dtype)
    zero = g.integers(5, 11, (n, m)).astype(np.uint8) if zeros else np.full((n, m), 8, np.uint8)
    wide = lambda v: np.repeat(v, group, axis=1)[:, :k].astype(np.float64)  # noqa: E731
    return x, code, scale, zero, (code - wide(zero)) * wide(scale)


def experts(v, k, name, held=lambda h: h):
    """y of the experts; `held`: how the inner activations are."""
    e = len(v["wr"])
    f, o = len(v["wg"]) // e, len(v["wd"]) // e
    index, share = V.route(v["x"], v["wr"], k, True)
    y = np.zeros((len(v["x"]), o))
    for i in range(e):
        at, slot = np.nonzero(index == i)
        if len(at):
            of = lambda w, n: v[w][i * n:(i + 1) * n].T  # noqa: E731
            h = U.act(name, v["x"][at] @ of("wg", f))[0] * (v["x"][at] @ of("wu", f))
            y[at] += share[at, slot][:, None] * (held(h) @ of("wd", o))
    return y
