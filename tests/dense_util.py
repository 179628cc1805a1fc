"""The dense operators restated in 64 bits, for their tests: 16-bit types as numpy holds them, dropout's mask, the block's
formulas and how far a kernel that follows them may be off."""
import numpy as np

from b2ctrain_amd import _native, nn

UNIT = {nn.BF16: 2.0 ** -8, nn.F16: 2.0 ** -11, nn.F32: 2.0 ** -24}  # largest relative rounding error
F32_SUM = 2.0 ** -24


def bf16_bits(x):
    """float32 -> bfloat16 bit patterns, to nearest even (finite and infinite values; NaN stays one)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def store(x, dtype):
    """The array that holds x's values in `dtype`."""
    if dtype == nn.F32:
        return np.ascontiguousarray(x, np.float32)
    if dtype == nn.F16:
        return np.ascontiguousarray(x, np.float16)
    return bf16_bits(np.asarray(x, np.float32))


def value(a, dtype):
    """The float64 values of a stored array."""
    if dtype == nn.BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rounded(x, dtype):
    return value(store(x, dtype), dtype)


class Held:
    """A matrix on the device inside a larger buffer: rows `cols + pad` apart, `shift` elements off the buffer's start. What
    surrounds it is filled, and checked by around()."""

    def __init__(self, x, dtype, pad=0, shift=0, rows=None, cols=None):
        self.dtype = dtype
        self.rows, self.cols = (rows, cols) if x is None else x.shape
        self.ld, self.shift = self.cols + pad, shift
        n = max(1, self.rows * self.ld + shift + 8)
        if dtype == nn.I8:
            flat = np.full(n, 113, np.int8)
        else:
            flat = store(np.full(n, 1.5e4), dtype)
        if x is not None:
            self._window(flat)[:] = x if dtype == nn.I8 else store(x, dtype)
        self.before, self.np_type = flat, flat.dtype
        self.dev = _native.DeviceArray(flat)
        self.matrix = nn.Matrix(self.dev.ptr + shift * flat.itemsize, self.rows, self.cols, self.ld, dtype, keep=self.dev)

    def _window(self, flat):
        return flat[self.shift:self.shift + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def get(self):
        flat = self.dev.download(self.np_type, self.before.shape)
        got = self._window(flat).copy()
        self._window(flat)[:] = self._window(self.before)
        assert np.array_equal(flat, self.before), "values around the matrix changed"
        return got.astype(np.int64) if self.dtype == nn.I8 else value(got, self.dtype)


class Space:
    """Workspace with a filled rim: what a plan asks for, to the byte, and nothing beyond it touched."""

    def __init__(self):
        self.held = []

    def __call__(self, n):
        flat = np.full(n + 256, 0xFF, np.uint8)  # every 16- and 32-bit float in it is a NaN
        dev = _native.DeviceArray(flat)
        self.held.append((dev, n))
        return dev

    def check(self):
        for dev, n in self.held:
            rim = dev.download(np.uint8, (n + 256,))[n:]
            assert (rim == 0xFF).all(), "a kernel wrote beyond its workspace"


def philox(counter, key):
    """Philox4x32-10: [n][4] counter words and two key words -> [n][4] words."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1).astype(np.uint32)


def threshold(p):
    return int(np.floor(float(np.float32(p)) * 65536 + 0.5))


def mask(rows, cols, p, seed, stream):
    """Dropout's factor of each value: 0, or 65536 / (65536 - T)."""
    n, t = rows * cols, threshold(p)
    g = np.arange(-(-n // 8), dtype=np.uint64)
    c = np.zeros((len(g), 4), np.uint64)
    c[:, 0], c[:, 1] = g & np.uint64(0xFFFFFFFF), g >> np.uint64(32)
    c[:, 2], c[:, 3] = stream & 0xFFFFFFFF, stream >> 32
    w = philox(c, (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([w & 0xFFFF, w >> 16], axis=2).reshape(-1)[:n]
    return np.where(bits >= t, 65536.0 / (65536 - t), 0.0).reshape(rows, cols)


_erf = None


def act(name, g):
    """The activation and its derivative."""
    global _erf
    if name == "relu":
        return np.maximum(g, 0), (g > 0).astype(np.float64)
    if name == "silu":
        s = 1 / (1 + np.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if _erf is None:
        from scipy.special import erf as _erf
    phi = 0.5 * (1 + _erf(g / np.sqrt(2)))
    return g * phi, phi + g * np.exp(-g * g / 2) / np.sqrt(2 * np.pi)


# Bounds of |act'| and |act''| over the line: silu 1.0998 and 1/2, gelu 1.1290 and 2 / sqrt(2 pi), relu 1 and (a rounded g
# keeps its sign) 0.
SLOPE = {"silu": 1.1, "gelu": 1.13, "relu": 1.0}
CURVE = {"silu": 0.5, "gelu": 0.8, "relu": 0.0}
ACT_EPS = 2.0 ** -20  # the activation itself, evaluated in single precision


def block(x, wg, wu, wd, name, r=None, m=1.0):
    g, u = x @ wg.T, x @ wu.T
    a, _ = act(name, g)
    y = ((a * u) @ wd.T) * m
    return y if r is None else y + r


def block_grads(x, wg, wu, wd, name, dy, m=1.0):
    g, u = x @ wg.T, x @ wu.T
    a, d = act(name, g)
    dz = dy * m
    dh = dz @ wd
    dg, du = dh * u * d, dh * a
    return {"dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dz.T @ (a * u)}


def block_bound(x, wg, wu, wd, name, dtype, r=None, m=1.0):
    """How far y may be off: sums of n products in single precision are off by (n + 8) 2^-24 of the sum of magnitudes; h is
    rounded once, y once."""
    e, b = UNIT[dtype], lambda n: (n + 8) * F32_SUM
    g, u = x @ wg.T, x @ wu.T
    a, _ = act(name, g)
    eg, eu = b(x.shape[1]) * (abs(x) @ abs(wg).T), b(x.shape[1]) * (abs(x) @ abs(wu).T)
    eh = SLOPE[name] * eg * (abs(u) + eu) + abs(a) * eu + (e + ACT_EPS) * abs(a * u) + ACT_EPS * abs(u)
    y = block(x, wg, wu, wd, name, r, m)
    return (eh @ abs(wd).T + b(wd.shape[1]) * (abs(a * u) @ abs(wd).T)) * m * 1.001 + e * abs(y) + 2.0 ** -24


def grads_bound(x, wg, wu, wd, name, dtype, dy, m=1.0, out=None):
    """The same of the gradients: g and u come back rounded, h, dg and du are rounded, and each output (`out`: its type)."""
    e, b = UNIT[dtype], lambda n: (n + 8) * F32_SUM
    eo = UNIT[dtype if out is None else out]
    M, D = x.shape
    F, O = wg.shape[0], wd.shape[0]
    g, u = x @ wg.T, x @ wu.T
    a, d = act(name, g)
    dz = dy * m
    dh = dz @ wd
    eg, eu = b(D) * (abs(x) @ abs(wg).T) + e * abs(g), b(D) * (abs(x) @ abs(wu).T) + e * abs(u)
    edh = b(O) * (abs(dz) @ abs(wd))
    ea, ed = SLOPE[name] * eg + ACT_EPS * (abs(a) + 1), CURVE[name] * eg + ACT_EPS * 4
    if name == "relu":  # a g within its error of zero may take either slope
        ed = ed + (abs(g) <= b(D) * (abs(x) @ abs(wg).T))
    eh = ea * (abs(u) + eu) + abs(a) * eu + e * abs(a * u)
    edg = (abs(dh) + edh) * ((abs(u) + eu) * ed + eu * abs(d)) + edh * abs(u * d) + e * abs(dh * u * d)
    edu = (abs(dh) + edh) * ea + edh * abs(a) + e * abs(dh * a)
    ref = block_grads(x, wg, wu, wd, name, dy, m)
    dg, du, tiny = dh * u * d, dh * a, 1e-7 if dtype == nn.F16 else 2.0 ** -24
    got = {"dx": edg @ abs(wg) + edu @ abs(wu) + b(2 * F) * (abs(dg) @ abs(wg) + abs(du) @ abs(wu)),
           "dw_gate": edg.T @ abs(x) + b(M) * (abs(dg).T @ abs(x)), "dw_up": edu.T @ abs(x) + b(M) * (abs(du).T @ abs(x)),
           "dw_down": abs(dz).T @ eh + b(M) * (abs(dz).T @ abs(a * u))}
    # values of fewer than 16 bits' normal range lose up to `tiny` when they are rounded, and so do the products of them
    small = {"dx": tiny * (abs(wg).sum(0) + abs(wu).sum(0) + 1)[None, :], "dw_gate": tiny * (abs(x).sum(0) + 1)[None, :],
             "dw_up": tiny * (abs(x).sum(0) + 1)[None, :], "dw_down": tiny * (abs(dz).sum(0) + 1)[:, None]}
    return ref, {k: got[k] * 1.01 + (eo if k != "dx" else e) * abs(ref[k]) + small[k] for k in got}


def quantised(x):
    """(values, scales) of rows in 8 bits, in single precision as the kernels do it."""
    x = np.asarray(x, np.float32)
    top = abs(x).max(axis=1)
    s = (top / np.float32(127)).astype(np.float32)
    safe = np.where(s > 0, s, np.float32(1))
    q = np.where(s[:, None] > 0, np.rint(x / safe[:, None]), 0).astype(np.float32)
    return np.clip(q, -127, 127).astype(np.int8), s
