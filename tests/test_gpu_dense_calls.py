"""Calls of the dense operators that differ from the usual ones in one thing: an alignment, a buffer's place, a size at the end of
its range; against their restatement in 64 bits (dense_util.py)."""
import ctypes as C

import numpy as np
import pytest

from b2ctrain_amd import _native, nn
from tests import dense_bounds as B
from tests import dense_util as U
from tests.gpu_harness import emit
from tests.test_gpu_dense import check_block, close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def i8_block(x, ws, ss, name, act_eps=2.0 ** -20):
    """y of the 8-bit block, and how far it may move by values of h that lie within single precision's rounding of the middle between two
    steps: each by one step of its row. act_eps: how far the activation may be off, beside 2^-20 of itself."""
    dense = lambda q, s, w, sw: (q.astype(np.float64) @ w.T.astype(np.float64)) * s[:, None].astype(np.float64) * sw[:, 0].astype(np.float64)  # noqa: E731
    q, sx = U.quantised(x)
    up = dense(q, sx, ws[1], ss[1])
    h = U.act(name, dense(q, sx, ws[0], ss[0]))[0] * up
    top = abs(h).max(axis=1, keepdims=True)
    step = top / 127
    safe = np.where(step > 0, step, 1)
    t = np.where(step > 0, h / safe, 0)
    unsure = abs(t - np.floor(t) - 0.5) <= (2.0 ** -20 * (abs(h) + top) + act_eps * abs(up)) / safe
    want = (np.rint(t) @ ws[2].T.astype(np.float64)) * step * ss[2][:, 0].astype(np.float64)
    return want, (unsure @ abs(ws[2]).T.astype(np.float64)) * step * ss[2][:, 0]


@pytest.mark.parametrize("rows,di,f,do,pad", [(64, 144, 256, 144, 0), (64, 256, 320, 256, 16), (200, 48, 1040, 48, 0), (20, 144, 256, 144, 0)])
@pytest.mark.parametrize("gate,up,down", [(0, 8, 0), (8, 0, 0), (8, 3, 8), (0, 0, 5)])
def test_i8_block_of_weights_aligned_differently(rows, di, f, do, pad, gate, up, down):
    emit(f"i8 block {rows} x {di}-{f}-{do} pad {pad}, weights {gate}, {up}, {down} bytes off")
    g = np.random.default_rng(rows + di)
    x = U.rounded(g.standard_normal((rows, di)), BF16)
    ws = [g.integers(-127, 128, s).astype(np.int8) for s in ((f, di), (f, di), (do, f))]
    ss = [(np.exp(g.uniform(-0.5, 0.5, (n, 1))) / 73 / np.sqrt(k)).astype(np.float32) for n, k in ((f, di), (f, di), (do, f))]
    hx, y, space = U.Held(x, BF16), U.Held(None, BF16, rows=rows, cols=do), U.Space()
    hw, hs = [U.Held(w, nn.I8, pad, shift) for w, shift in zip(ws, (gate, up, down))], [U.Held(s, F32) for s in ss]
    nn.I8FeedForward(hx.matrix, hw[0].matrix, hs[0].matrix, hw[1].matrix, hs[1].matrix, hw[2].matrix, hs[2].matrix, y.matrix, room=space).run()
    want, slack = i8_block(x, ws, ss, "silu")
    close("y", y.get(), want, (U.UNIT[BF16] + 2.0 ** -19) * abs(want) + slack + 1e-30)
    space.check()


class Handle:
    """A b2c_dense handle with the C entries that the tests call."""

    def __init__(self):
        self.L = _native.lib()
        for name, args in (("b2c_feed_forward", [C.c_void_p, C.POINTER(nn.FfnArgs), C.c_int, C.c_void_p]),
                           ("b2c_feed_forward_backward", [C.c_void_p, C.POINTER(nn.FfnGradArgs), C.c_void_p])):
            getattr(self.L, name).argtypes = args
        self.L.b2c_dense_create.restype = C.c_void_p
        self.L.b2c_dense_destroy.argtypes = [C.c_void_p]
        self.ptr = self.L.b2c_dense_create()

    def forward(self, ff, train=1):
        return self.L.b2c_feed_forward(self.ptr, C.byref(ff.args), train, None)

    def backward(self, ff):
        return self.L.b2c_feed_forward_backward(self.ptr, C.byref(ff.grad), None)

    def close(self):
        self.L.b2c_dense_destroy(self.ptr)


def test_a_handle_refuses_gradients_of_another_forward_pass():
    """What the handle kept is of one call: gradients of smaller sizes, another type, activation or mask are refused, though they
    would fit what is there."""
    g = np.random.default_rng(1)
    space, held, d = U.Space(), [], Handle()

    def block(rows, di=200, f=330, dtype=BF16, **kw):
        h = [U.Held(g.standard_normal(s) * 0.1, dtype) for s in ((rows, di), (f, di), (f, di), (di, f), (rows, di))]
        out = [U.Held(None, dtype, rows=a, cols=b) for a, b in ((rows, di), (rows, di), (f, di))]
        held.extend(h + out)
        x, wg, wu, wd, dy = (m.matrix for m in h)
        y, dx, dw = (m.matrix for m in out)
        ff = nn.FeedForward(x, wg, wu, wd, y, **{"p": 0.2, "seed": 3, "train": True, "room": space, **kw})
        ff.gradients(dy, dx=dx, dw_gate=dw, room=space)
        return ff

    try:
        large = block(300)
        others = {"rows": block(100), "d_hidden": block(300, f=320), "d_in": block(300, di=190), "type": block(300, dtype=F16),
                  "act": block(300, act="gelu"), "p": block(300, p=0.3), "seed": block(300, seed=4), "stream id": block(300, stream_id=9)}
        assert d.backward(large) != 0 and b"no forward pass" in d.L.b2c_last_error()
        assert d.forward(large) == 0 and d.backward(large) == 0 and d.backward(large) == 0
        for what, other in others.items():
            emit(f"gradients with another {what}")
            assert d.backward(other) != 0 and b"no forward pass" in d.L.b2c_last_error(), what
        assert d.forward(others["rows"], train=0) == 0 and d.backward(large) == 0  # answers leave what is kept alone
        wrong = nn.FfnArgs.from_buffer_copy(large.args)
        wrong.act = 17
        assert d.L.b2c_feed_forward(d.ptr, C.byref(wrong), 1, None) != 0
        assert d.backward(large) != 0 and b"no forward pass" in d.L.b2c_last_error()  # the last pass to be kept was refused
        assert d.forward(others["rows"]) == 0 and d.backward(others["rows"]) == 0
        plain, again = block(50, p=0.0), block(50, p=0.0, seed=8, stream_id=2)  # without dropout there is no mask to differ
        assert d.forward(plain) == 0 and d.backward(again) == 0
    finally:
        d.close()
    space.check()


def subnormal_rows(cols):
    """Rows whose largest magnitude is some units of 2^-149, the smallest single-precision value: their scale is so coarse that the
    quotient may pass 127."""
    tops = [1, 63, 64, 100, 127, 128, 160, 190, 191, 500, 15811, 16065, 16066, 1 << 20]
    g = np.random.default_rng(cols)
    bits = (g.uniform(0, 1, (len(tops), cols)) * (np.array(tops)[:, None] + 1)).astype(np.uint32)
    bits[:, 0] = tops
    bits[:, -1] = tops
    x = bits.view(np.float32)
    x[:, -1] *= -1
    return x


@pytest.mark.parametrize("cols", [7, 64, 200, 1100, 5000])
@pytest.mark.parametrize("copies", [1, 200])
def test_quantize_rows_of_subnormals(cols, copies):
    emit(f"quantize {copies} times 14 x {cols} subnormals")
    x = np.tile(subnormal_rows(cols), (copies, 1))
    h, q, s = U.Held(x, F32), U.Held(None, nn.I8, rows=len(x), cols=cols), U.Held(None, F32, rows=len(x), cols=1)
    nn.QuantizeRows(h.matrix, q.matrix, s.matrix).run()
    want, scale = U.quantised(x)  # held to -127 .. 127
    assert np.array_equal(s.get()[:, 0], scale) and np.array_equal(q.get(), want)


@pytest.mark.parametrize("rows,di,do", [(7, 64, 32), (14, 3000, 32), (70, 64, 32), (70, 200, 40)])
def test_i8_linear_of_subnormals(rows, di, do):
    """One layer's ways with a row: in the product, in registers, before the tiles. y = acc sx sw is off by its products in single
    precision, the first of which may be subnormal: half of 2^-149, times sw."""
    emit(f"i8 linear {rows} x {di}-{do} of subnormals")
    x = np.resize(subnormal_rows(di)[::-1], (rows, di))
    w, sw = np.random.default_rng(do).integers(-127, 128, (do, di)).astype(np.int8), np.float32(2.0 ** 100)
    hx, hw, hs, y, space = U.Held(x, F32), U.Held(w, nn.I8), U.Held(np.full((do, 1), sw), F32), U.Held(None, F32, rows=rows, cols=do), U.Space()
    nn.I8Linear(hx.matrix, hw.matrix, hs.matrix, y.matrix, room=space).run()
    q, sx = U.quantised(x)
    want = (q.astype(np.float64) @ w.T.astype(np.float64)) * sx[:, None].astype(np.float64) * float(sw)
    close("y", y.get(), want, 4 * 2.0 ** -24 * abs(want) + 2.0 ** -150 * float(sw) * 1.001)
    space.check()


@pytest.mark.parametrize("rows,di,f,do", [(40, 64, 128, 64), (70, 100, 300, 72), (20, 64, 128, 64), (70, 200, 300, 72)])
@pytest.mark.parametrize("name", ["silu", "relu"])
@pytest.mark.parametrize("gate", [1e-28, 1e-31, 1e-33])
def test_i8_block_with_tiny_inner_activations(rows, di, f, do, name, gate):
    """h far below one, brought back by the down weights' scales: 8 bits of a row go by its own largest value, however small. Near
    zero both activations are off by their relative error alone."""
    emit(f"i8 block {rows} x {di}-{f}-{do} {name}, gate scales of {gate}")
    g = np.random.default_rng(rows + di)
    x = g.standard_normal((rows, di)).astype(np.float32)
    x[5] = 0
    ws = [g.integers(-127, 128, s).astype(np.int8) for s in ((f, di), (f, di), (do, f))]
    ss = [(np.exp(g.uniform(-0.5, 0.5, (n, 1))) * k).astype(np.float32) for n, k in ((f, gate / 73), (f, 1 / 73), (do, 1e-3 / gate))]
    hx, y, space = U.Held(x, F32), U.Held(None, F32, rows=rows, cols=do), U.Space()
    hw, hs = [U.Held(w, nn.I8) for w in ws], [U.Held(s, F32) for s in ss]
    nn.I8FeedForward(hx.matrix, hw[0].matrix, hs[0].matrix, hw[1].matrix, hs[1].matrix, hw[2].matrix, hs[2].matrix, y.matrix, act=name,
                     room=space).run()
    want, slack = i8_block(x, ws, ss, name, 0)
    got = y.get()
    assert (got[5] == 0).all()
    close("y", got, want, 2.0 ** -18 * abs(want) + slack + 1e-30)
    space.check()


class Raw:
    """Device memory that is not filled, with windows of it to write and read."""

    hip = None

    def __init__(self, values, np_type):
        Raw.hip = Raw.hip or C.CDLL("libamdhip64.so.7")  # the library's own copy
        self.type, self.ptr = np.dtype(np_type), C.c_void_p()
        free, total = C.c_size_t(), C.c_size_t()
        self.check(self.hip.hipMemGetInfo(C.byref(free), C.byref(total)))
        if free.value < values * self.type.itemsize + (1 << 30):
            pytest.skip(f"needs {values * self.type.itemsize >> 30} GiB of device memory")
        self.check(self.hip.hipMalloc(C.byref(self.ptr), C.c_size_t(values * self.type.itemsize)))

    @staticmethod
    def check(rc):
        assert rc == 0, f"hipError {rc}"

    def at(self, first):
        return C.c_void_p(self.ptr.value + first * self.type.itemsize)

    def write(self, first, x):
        x = np.ascontiguousarray(x, self.type)
        self.check(self.hip.hipMemcpy(self.at(first), x.ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), 1))

    def read(self, first, n):
        x = np.empty(n, self.type)
        self.check(self.hip.hipMemcpy(x.ctypes.data_as(C.c_void_p), self.at(first), C.c_size_t(x.nbytes), 2))
        return x

    def free(self):
        self.hip.hipFree(self.ptr)


def test_quantize_rows_of_more_rows_than_a_launch_has_threads():
    rows, n = (1 << 30) + 1003, 1000
    emit(f"quantize {rows} x 1, 7 GB")
    x, q, s = Raw(rows, np.float16), Raw(rows, np.int8), Raw(rows, np.float32)
    try:
        g = np.random.default_rng(1)
        parts = {first: g.standard_normal((n, 1)).astype(np.float16) for first in (0, (1 << 30) - 500, rows - n)}
        for first, v in parts.items():
            x.write(first, v)
        nn.QuantizeRows(nn.Matrix(x.ptr.value, rows, 1, 1, F16), nn.Matrix(q.ptr.value, rows, 1, 1, nn.I8), nn.Matrix(s.ptr.value, rows, 1, 1, F32)).run()
        for first in (rows - n, 0):
            want, scale = U.quantised(parts[first])
            assert np.array_equal(q.read(first, n), want[:, 0]) and np.array_equal(s.read(first, n), scale), first
    finally:
        for m in (x, q, s):
            m.free()


@pytest.mark.parametrize("rows,cols,ld", [(1, (1 << 31) - 1, (1 << 31) - 1), ((1 << 24) + 1, 2049, 2049), ((1 << 24) + 1, 2049, 2050)])
def test_dropout_of_more_values_than_a_launch_has_threads(rows, cols, ld):
    """In place, windows at the start, around the value that the 2^32nd thread takes, and at the end."""
    emit(f"dropout {rows} x {cols}, rows {ld} apart, {rows * ld / 2 ** 29:.0f} GiB")
    p, seed, stream = 0.3, 11, 12
    x = Raw(rows * ld, np.float16)
    try:
        places = sorted({0, min(rows // 2, (1 << 35) // cols), rows - 1})
        parts = {m: np.random.default_rng(m).standard_normal(min(cols, 5000)).astype(np.float16) for m in places}
        for m, v in parts.items():
            x.write(m * ld + cols - len(v), v)
        h = nn.Matrix(x.ptr.value, rows, cols, ld, F16)
        nn.Dropout(h, h, p, seed, stream).run()
        for m, v in parts.items():
            e = m * cols + cols - len(v)
            first = e // 8 * 8
            want = U.value(v, F16) * window(first, e + len(v), p, seed, stream)[e - first:]
            close(f"y of row {m}", U.value(x.read(m * ld + cols - len(v), len(v)), F16), want,
                  U.UNIT[F16] * abs(want) + 3 * 2.0 ** -24 * abs(want) + 2.0 ** -25)
    finally:
        x.free()


def window(first, end, p, seed, stream):
    """Dropout's factors of values first .. end - 1, `first` a multiple of 8."""
    at = np.arange(first // 8, -(-end // 8), dtype=np.uint64)
    c = np.zeros((len(at), 4), np.uint64)
    c[:, 0], c[:, 1] = at & np.uint64(0xFFFFFFFF), at >> np.uint64(32)
    c[:, 2], c[:, 3] = stream & 0xFFFFFFFF, stream >> 32
    w = U.philox(c, (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([w & 0xFFFF, w >> 16], axis=2).reshape(-1)[:end - first]
    t = U.threshold(p)
    return np.where(bits >= t, 65536.0 / (65536 - t), 0.0)


@pytest.mark.parametrize("sizes", [(16384, 33, 72, 24), (16399, 64, 256, 64), (17001, 128, 96, 16), (16384, 7, 200, 3), (16500, 61, 130, 128),
                                   (33000, 32, 512, 32)])
@pytest.mark.parametrize("dtype,name,p,residual,pad,shift", [(BF16, "silu", 0.0, False, 0, 0), (F16, "gelu", 0.2, True, 5, 1),
                                                             (BF16, "relu", 0.1, True, 8, 0)])
def test_heads(sizes, dtype, name, p, residual, pad, shift):
    """Narrow blocks of as many rows as their own kernels are for."""
    check_block(*sizes, dtype, name, p, residual, pad, shift)


@pytest.mark.parametrize("sizes", [(98304 + 77, 24, 40, 16), (100_001, 64, 90, 48), (98304, 128, 33, 100)])
def test_heads_of_two_row_tiles_a_wave(sizes):
    check_block(*sizes, BF16, "silu", 0.1, True, 0, 0)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("sizes", [(16384, 40, 72, 24), (16385, 100, 300, 64)])
def test_heads_with_weight_gradients_in_single_precision(sizes, accumulate):
    check_block(*sizes, BF16, "silu", 0.1, False, 0, 0, grad=F32, accumulate=accumulate)


@pytest.mark.parametrize("sizes", [(40, 96, 8192, 96), (256, 128, 2048, 128), (2000, 64, 1030, 33), (100, 64, 64, 64), (65, 96, 65, 3)])
@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu")])
def test_narrow_blocks_of_few_rows(sizes, dtype, name):
    check_block(*sizes, dtype, name, 0.2, True, 0, 0)


@pytest.mark.parametrize("sizes", B.SINGLE + [(16384, 40, 1, 24), (16384, 128, 1, 100), (40, 24, 1, 16), (40, 96, 1, 128)])
@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu"), (BF16, "relu")])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_gradients_have_no_other_roundings(sizes, dtype, name, p):
    rows, di, f, do = sizes
    emit(f"gradients of {rows} x {di}-{f}-{do} type {dtype} {name} p {p}")
    x, wg, wu, wd, dy = B.make(*sizes, dtype, rows + f)
    space, y = U.Space(), U.Held(None, dtype, rows=rows, cols=do)
    h = [U.Held(v, dtype) for v in (x, wg, wu, wd, dy)]
    ff = nn.FeedForward(*(v.matrix for v in h[:4]), y.matrix, act=name, p=p, seed=7, stream_id=5, train=True, room=space)
    out = {k: U.Held(None, dtype, rows=a, cols=b) for k, a, b in (("dx", rows, di), ("dw_gate", f, di), ("dw_up", f, di), ("dw_down", do, f))}
    ff.gradients(h[4].matrix, **{k: o.matrix for k, o in out.items()}, room=space)
    ff.forward()
    ff.backward()
    m = U.mask(rows, do, p, 7, 5) if p else np.ones((rows, do))
    ref, bound = B.grads_bound(x, wg, wu, wd, name, dtype, dy, m)
    for k, o in out.items():
        close(k, o.get(), ref[k], bound[k])
    space.check()
