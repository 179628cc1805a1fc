"""The dense operators on the GPU against their restatement in 64 bits (dense_util.py), which also says how far a kernel that
sums in single precision and rounds where the documentation says may be off, value by value."""
import ctypes as C

import numpy as np
import pytest

from b2ctrain_amd import _native, nn
from tests import dense_util as U
from tests.gpu_harness import emit

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def close(name, got, want, bound):
    off = np.abs(got - want) - bound
    i = np.unravel_index(np.argmax(off), off.shape) if off.size else None
    assert not off.size or (np.isfinite(got).all() and off[i] <= 0), \
        f"{name}{list(i)}: {got[i]} is {abs(got[i] - want[i]):.3g} from {want[i]}, allowed {bound[i]:.3g}"


def sync(stream=None):
    _native.DeviceArray(np.zeros(4, np.float32)).download(np.float32, (4,))  # the default stream's synchronous copy


# ---- dropout -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,pad,shift,p", [
    (1, 1, 0, 0, 0.5), (1, 7, 0, 0, 0.5), (3, 8, 0, 0, 0.25), (64, 64, 0, 0, 0.1), (37, 45, 0, 0, 0.25), (37, 45, 3, 1, 0.25),
    (129, 16, 8, 0, 0.9), (5, 1000, 24, 3, 0.0), (300, 257, 0, 1, 0.3), (2000, 3, 0, 0, 0.6), (1, 70001, 0, 0, 0.1)])
def test_dropout(dtype, rows, cols, pad, shift, p):
    emit(f"dropout {rows}x{cols} pad {pad} shift {shift} type {dtype} p {p}")
    g = np.random.default_rng(rows * 1000 + cols)
    seed, stream = 0x9E3779B97F4A7C15, (1 << 63) + 12345
    x, r = U.rounded(g.standard_normal((rows, cols)), dtype), U.rounded(g.standard_normal((rows, cols)), dtype)
    m = U.mask(rows, cols, p, seed, stream)
    for residual in (False, True):
        hx, hr = U.Held(x, dtype, pad, shift), U.Held(r, dtype, pad, shift)
        y = U.Held(None, dtype, pad, shift, rows, cols)
        nn.Dropout(hx.matrix, y.matrix, p, seed, stream, residual=hr.matrix if residual else None).run()
        want = x * m + (r if residual else 0)
        # the scale, the product and the sum are rounded in single precision, the result once to its type
        bound = U.UNIT[dtype] * abs(want) + 3 * 2.0 ** -24 * (abs(x * m) + abs(r) * residual) + 2.0 ** -25 * (dtype == F16)
        got = y.get()
        close("y", got, want, bound)
        assert residual or np.array_equal(got != 0, (m > 0) & (got != 0)) and np.array_equal(got[m == 0], np.zeros((m == 0).sum()))
        nn.Dropout(hx.matrix, hx.matrix, p, seed, stream, residual=hr.matrix if residual else None).run()  # in place
        assert np.array_equal(hx.get(), got)


def test_dropout_drops_what_is_not_finite():
    x = np.tile(np.array([[np.inf, -np.inf, np.nan, 1.0]]), (32, 4))
    m = U.mask(32, 16, 0.5, 3, 4)
    h, y = U.Held(x, F32), U.Held(None, F32, rows=32, cols=16)
    nn.Dropout(h.matrix, y.matrix, 0.5, 3, 4).run()
    got = y.get()
    assert (got[m == 0] == 0).all()
    assert np.array_equal(got[m > 0], (x * 2)[m > 0], equal_nan=True)


# ---- the block ---------------------------------------------------------------------------------------------

SIZES = [  # rows, d_in, d_hidden, d_out
    (1, 1, 1, 1), (1, 64, 128, 64), (3, 17, 5, 9), (16, 96, 256, 96), (17, 33, 64, 40), (32, 512, 100, 48), (33, 40, 72, 24),
    (64, 64, 64, 64), (100, 7, 200, 3), (129, 200, 330, 136), (257, 64, 256, 64), (300, 128, 96, 16), (1000, 24, 40, 72),
    (63, 1032, 70, 520)]


def make(rows, di, f, do, dtype, seed, pad, shift):
    g = np.random.default_rng(seed)
    q = lambda *s, k=1.0: U.rounded(g.standard_normal(s) * k, dtype)  # noqa: E731
    v = dict(x=q(rows, di), wg=q(f, di, k=di ** -0.5), wu=q(f, di, k=di ** -0.5), wd=q(do, f, k=f ** -0.5), r=q(rows, do),
             dy=q(rows, do, k=0.3))
    return v, {k: U.Held(a, dtype, pad, shift) for k, a in v.items()}


def check_block(rows, di, f, do, dtype, name, p, residual, pad, shift, grad=None, accumulate=False, seed=0, sample=None):
    emit(f"block {rows} x {di}-{f}-{do} type {dtype} {name} p {p} pad {pad} shift {shift}")
    v, h = make(rows, di, f, do, dtype, seed + rows, pad, shift)
    key, stream = 77 + seed, 5
    m = U.mask(rows, do, p, key, stream) if p else np.ones((rows, do))
    args = [v[k] for k in ("x", "wg", "wu", "wd")]
    r = v["r"] if residual else None
    space = U.Space()
    grad = dtype if grad is None else grad
    for train in (False, True):
        y = U.Held(None, dtype, pad, shift, rows, do)
        ff = nn.FeedForward(h["x"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, act=name,
                            residual=h["r"].matrix if residual else None, p=p, seed=key, stream_id=stream, train=train, room=space)
        ff.forward()
        close("y", y.get(), U.block(*args, name, r, m), U.block_bound(*args, name, dtype, r, m))
    out = {"dx": U.Held(None, dtype, pad, shift, rows, di)}
    start = np.random.default_rng(3).standard_normal((max(f, do), max(di, f)))
    for k, (a, b) in (("dw_gate", (f, di)), ("dw_up", (f, di)), ("dw_down", (do, f))):
        out[k] = U.Held(U.rounded(start[:a, :b], grad) if accumulate else None, grad, pad, shift, a, b)
    ff.gradients(h["dy"].matrix, **{k: o.matrix for k, o in out.items()}, accumulate=accumulate, room=space)
    ff.backward()
    ref, bound = U.grads_bound(*args, name, dtype, v["dy"], m, out=grad)
    got = {k: o.get() for k, o in out.items()}
    for k in out:
        add = U.rounded(start[:ref[k].shape[0], :ref[k].shape[1]], F32) if accumulate and k != "dx" else 0
        close(k, got[k], ref[k] + add, bound[k] + 2.0 ** -23 * abs(ref[k] + add) * (k != "dx" and grad == F32))
    space.check()
    return ff, out, got


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu"), (F16, "relu")])
def test_block(sizes, dtype, name):
    check_block(*sizes, dtype, name, 0.0, False, 0, 0)


@pytest.mark.parametrize("sizes", [(1, 64, 128, 64), (5, 24, 40, 16), (33, 40, 72, 24), (129, 200, 330, 136), (257, 64, 256, 64), (300, 61, 200, 63)])
@pytest.mark.parametrize("dtype,name", [(BF16, "gelu"), (F16, "silu"), (BF16, "relu")])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (5, 1), (0, 3)])
def test_block_dropout_residual_strides(sizes, dtype, name, pad, shift):
    check_block(*sizes, dtype, name, 0.2, True, pad, shift)


@pytest.mark.parametrize("sizes", [(33, 40, 72, 24), (257, 64, 256, 64), (2100, 64, 32, 64)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_block_weight_gradients_in_single_precision(sizes, accumulate):
    check_block(*sizes, BF16, "silu", 0.1, False, 0, 0, grad=F32, accumulate=accumulate)


@pytest.mark.parametrize("sizes", [(700, 600, 1100, 520), (2048, 768, 1024, 768), (9000, 136, 200, 72), (6000, 32, 512, 128), (4100, 128, 384, 128)])
def test_block_larger(sizes):
    """Large enough for every tile size and for sums split over k."""
    check_block(*sizes, BF16, "silu", 0.1, True, 0, 0)


def test_block_largest_tiles():
    """Rows and columns picked from a block that fills the device with the largest tiles."""
    rows, di, f, do = 2304, 2048, 2304, 2048
    emit(f"block {rows} x {di}-{f}-{do}")
    v, h = make(rows, di, f, do, BF16, 1, 0, 0)
    y, space = U.Held(None, BF16, rows=rows, cols=do), U.Space()
    ff = nn.FeedForward(h["x"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, train=True, room=space)
    out = {k: U.Held(None, BF16, rows=a, cols=b) for k, a, b in (("dx", rows, di), ("dw_gate", f, di), ("dw_up", f, di), ("dw_down", do, f))}
    ff.gradients(h["dy"].matrix, **{k: o.matrix for k, o in out.items()}, room=space)
    ff.forward()
    ff.backward()
    pick = np.array([0, 1, 255, 256, 1000, rows - 1])
    args = [v[k] for k in ("x", "wg", "wu", "wd")]
    some = [v["x"][pick], *args[1:]]
    close("y", y.get()[pick], U.block(*some, "silu"), U.block_bound(*some, "silu", BF16))
    ref, bound = U.grads_bound(*some, "silu", BF16, v["dy"][pick])
    close("dx", out["dx"].get()[pick], ref["dx"], bound["dx"])
    hid = np.array([0, 127, 128, 2047, f - 1])  # rows of the gate's and up's gradients: a block of five hidden units
    ref, bound = U.grads_bound(v["x"], v["wg"][hid], v["wu"][hid], v["wd"][:, hid], "silu", BF16, v["dy"])
    close("dw_gate", out["dw_gate"].get()[hid], ref["dw_gate"], bound["dw_gate"])
    close("dw_up", out["dw_up"].get()[hid], ref["dw_up"], bound["dw_up"])
    close("dw_down", out["dw_down"].get()[:, hid], ref["dw_down"], bound["dw_down"])
    space.check()


def test_block_gradient_along_its_direction():
    """The forward kernel's own difference along the sign of the gradient: (L(x + e s) - L(x - e s)) / 2 e = sum |dx|. L is a sum
    of 512 x 64 rounded outputs; their rounding errors, of at most 2^-12 |y dy| each and independent, and e^2 stay below 2%."""
    rows, di, f, do, e = 512, 64, 128, 64, 2.0 ** -5
    ff, out, got = check_block(rows, di, f, do, F16, "silu", 0.2, False, 0, 0, seed=2)
    v, h = make(rows, di, f, do, F16, 2 + rows, 0, 0)
    x = v["x"]
    s = np.sign(got["dx"])
    loss = []
    for t in (e, -e):
        hx, y, space = U.Held(x + t * s, F16), U.Held(None, F16, rows=rows, cols=do), U.Space()
        nn.FeedForward(hx.matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, p=0.2, seed=79, stream_id=5, room=space).forward()
        loss.append(((y.get() * v["dy"]).sum(), U.rounded(x + t * s, F16)))
    step = ((loss[0][1] - loss[1][1]) * got["dx"]).sum()
    assert abs(loss[0][0] - loss[1][0] - step) < 0.02 * step


def test_block_in_place_residual_and_partial_gradients():
    rows, di, f, do = 70, 64, 96, 64
    v, h = make(rows, di, f, do, BF16, 9, 0, 0)
    space = U.Space()
    W = [h[k].matrix for k in ("wg", "wu", "wd")]
    y = U.Held(None, BF16, rows=rows, cols=do)
    nn.FeedForward(h["x"].matrix, *W, y.matrix, residual=h["r"].matrix, room=space).forward()
    both = U.Held(v["r"], BF16)
    nn.FeedForward(h["x"].matrix, *W, both.matrix, residual=both.matrix, room=space).forward()
    assert np.array_equal(y.get(), both.get())
    shapes = {"dx": (rows, di), "dw_gate": (f, di), "dw_up": (f, di), "dw_down": (do, f)}
    whole = {k: U.Held(None, BF16, rows=a, cols=b) for k, (a, b) in shapes.items()}
    ff = nn.FeedForward(h["x"].matrix, *W, y.matrix, train=True, room=space)
    ff.forward()
    ff.gradients(h["dy"].matrix, **{k: o.matrix for k, o in whole.items()}, room=space)
    ff.backward()
    want = {k: o.get() for k, o in whole.items()}
    for k, (a, b) in shapes.items():  # one at a time gives the same values
        one = U.Held(None, BF16, rows=a, cols=b)
        ff.gradients(h["dy"].matrix, **{k: one.matrix}, room=space)
        ff.backward()
        assert np.array_equal(one.get(), want[k]), k
    ff.gradients(h["dy"].matrix, room=space)
    ff.backward()
    space.check()


def test_no_rows_give_no_weight_gradient():
    f = U.Held(np.ones((24, 16)), BF16)
    d = U.Held(np.ones((16, 24)), BF16)
    x, y = nn.Matrix(0, 0, 16, 16, BF16), nn.Matrix(0, 0, 16, 16, BF16)
    space = U.Space()
    ff = nn.FeedForward(x, f.matrix, f.matrix, d.matrix, y, train=True, room=space)
    ff.forward()
    dw, dd = U.Held(np.ones((24, 16)), F32), U.Held(np.ones((16, 24)), F32)
    ff.gradients(y, dw_gate=dw.matrix, dw_down=dd.matrix, accumulate=True, room=space)
    ff.backward()
    assert (dw.get() == 1).all() and (dd.get() == 1).all()
    ff.gradients(y, dw_gate=dw.matrix, dw_down=dd.matrix, room=space)
    ff.backward()
    assert (dw.get() == 0).all() and (dd.get() == 0).all()


@pytest.mark.parametrize("sizes", [(40, 64, 128, 64), (9, 64, 128, 64), (300, 100, 90, 50)])
def test_block_keeps_a_bad_row_to_itself(sizes):
    rows, di, f, do = sizes
    v, h = make(rows, di, f, do, BF16, 4, 0, 0)
    space = U.Space()

    def run(x, dy):
        hx, hd, y, dx = U.Held(x, BF16), U.Held(dy, BF16), U.Held(None, BF16, rows=rows, cols=do), U.Held(None, BF16, rows=rows, cols=di)
        ff = nn.FeedForward(hx.matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, train=True, room=space)
        ff.gradients(hd.matrix, dx=dx.matrix, room=space)
        ff.forward()
        ff.backward()
        return y.get(), dx.get()

    x, dy = v["x"].copy(), v["dy"].copy()
    y0, dx0 = run(x, dy)
    x[3, 1], dy[5, 2] = np.nan, np.inf
    y1, dx1 = run(x, dy)
    assert np.isnan(y1[3]).all() and np.isnan(dx1[3]).all() and not np.isfinite(dx1[5]).all()
    keep = np.arange(rows) != 3
    assert np.array_equal(y0[keep], y1[keep])
    keep &= np.arange(rows) != 5
    assert np.array_equal(dx0[keep], dx1[keep])


def test_runs_repeat_bit_for_bit_on_a_stream():
    """Twice on a context's stream, in workspaces with other contents: the same bits."""
    rows, di, f, do = 3000, 128, 192, 128
    v, h = make(rows, di, f, do, BF16, 6, 0, 0)
    L = _native.lib()
    ctx = L.b2c_ctx_create()
    try:
        got = []
        for _ in range(2):
            space = U.Space()
            y = U.Held(None, BF16, rows=rows, cols=do)
            out = {k: U.Held(None, BF16, rows=a, cols=b) for k, a, b in (("dx", rows, di), ("dw_gate", f, di), ("dw_up", f, di), ("dw_down", do, f))}
            ff = nn.FeedForward(h["x"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, p=0.3, seed=1, train=True, room=space)
            ff.gradients(h["dy"].matrix, **{k: o.matrix for k, o in out.items()}, room=space)
            s = L.b2c_ctx_stream(ctx)
            ff.forward(s)
            ff.backward(s)
            assert L.b2c_ctx_synchronize(ctx) == 0
            got.append([y.get()] + [o.get() for o in out.values()])
            ff.set_stream_id(1)
            ff.forward(s)
            assert L.b2c_ctx_synchronize(ctx) == 0
            assert not np.array_equal(y.get(), got[-1][0])  # another mask
        assert all(np.array_equal(a, b) for a, b in zip(*got))
    finally:
        L.b2c_ctx_destroy(ctx)


class Graph:
    """What `work(stream)` launches, recorded once."""

    def __init__(self, stream, work):
        self.hip, self.stream, self.exec = C.CDLL("libamdhip64.so.7"), C.c_void_p(stream), C.c_void_p()  # the library's own copy
        graph = C.c_void_p()
        self.check(self.hip.hipStreamBeginCapture(self.stream, 1))  # this thread's calls
        work(stream)
        self.check(self.hip.hipStreamEndCapture(self.stream, C.byref(graph)))
        self.check(self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)))
        self.check(self.hip.hipGraphDestroy(graph))

    @staticmethod
    def check(rc):
        assert rc == 0, f"hipError {rc}"

    def replay(self):
        self.check(self.hip.hipGraphLaunch(self.exec, self.stream))
        self.check(self.hip.hipStreamSynchronize(self.stream))

    def close(self):
        self.check(self.hip.hipGraphExecDestroy(self.exec))


@pytest.mark.parametrize("rows,di,f,do,pad", [(5, 200, 100, 56, 0), (129, 200, 330, 136, 3), (3000, 64, 256, 64, 0), (300, 512, 1032, 512, 0)])
def test_a_recorded_step_replays(rows, di, f, do, pad):
    """Dropout, the block with its gradients and its 8-bit form from a recorded graph, between passes with another mask."""
    emit(f"graph {rows} x {di}-{f}-{do} pad {pad}")
    v, h = make(rows, di, f, do, BF16, 9, pad, 0)
    g, space = np.random.default_rng(rows), U.Space()
    x, y, z = [U.Held(None, BF16, pad, 0, rows, n) for n in (di, do, do)]
    out = {k: U.Held(None, BF16, pad, 0, a, b) for k, a, b in (("dx", rows, di), ("dw_gate", f, di), ("dw_up", f, di), ("dw_down", do, f))}
    drop = nn.Dropout(h["x"].matrix, x.matrix, 0.25, 3, 0)
    ff = nn.FeedForward(x.matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, p=0.3, seed=1, train=True, room=space)
    ff.gradients(h["dy"].matrix, **{k: o.matrix for k, o in out.items()}, room=space)
    hw = [U.Held(g.integers(-127, 128, s).astype(np.int8), nn.I8, pad) for s in ((f, di), (f, di), (do, f))]
    hs = [U.Held(np.full((n, 1), 0.01, np.float32), F32) for n in (f, f, do)]
    i8 = nn.I8FeedForward(x.matrix, hw[0].matrix, hs[0].matrix, hw[1].matrix, hs[1].matrix, hw[2].matrix, hs[2].matrix, z.matrix, room=space)

    def step(mask, stream):
        drop.set_stream_id(mask)
        ff.set_stream_id(mask)
        drop.run(stream)
        ff.forward(stream)
        ff.backward(stream)
        i8.run(stream)

    L = _native.lib()
    ctx = L.b2c_ctx_create()
    try:
        s = L.b2c_ctx_stream(ctx)
        results = lambda: [o.get() for o in (x, y, z, *out.values())]  # noqa: E731
        step(0, s)
        assert L.b2c_ctx_synchronize(ctx) == 0
        want = results()
        graph = Graph(s, lambda stream: step(0, stream))
        for _ in range(3):
            step(1, s)
            assert L.b2c_ctx_synchronize(ctx) == 0
            assert not any(np.array_equal(a, b) for a, b in zip(want, results()))
            graph.replay()
            assert all(np.array_equal(a, b) for a, b in zip(want, results()))
        graph.close()
    finally:
        L.b2c_ctx_destroy(ctx)
    space.check()


# ---- 8 bits ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,pad,shift,qpad", [(1, 1, 0, 0, 0), (5, 64, 0, 0, 0), (33, 100, 0, 0, 12), (64, 333, 7, 1, 3), (3, 4999, 0, 0, 9),
                                                     (2000, 64, 0, 0, 0), (700, 256, 0, 0, 0), (9, 20000, 0, 0, 0)])
def test_quantize_rows(dtype, rows, cols, pad, shift, qpad):
    emit(f"quantize {rows}x{cols} type {dtype} pad {pad}")
    g = np.random.default_rng(cols)
    x = U.rounded(g.standard_normal((rows, cols)) * np.exp(g.uniform(-6, 6, (rows, 1))), dtype)
    if rows > 4:
        x[1] = 0
        x[2, cols // 2], x[3, 0] = np.inf, np.nan
    hx = U.Held(x, dtype, pad, shift)
    q = _native.DeviceArray(np.full((rows, cols + qpad), 55, np.int8))
    s = U.Held(None, F32, rows=rows, cols=1)
    nn.QuantizeRows(hx.matrix, nn.Matrix(q.ptr, rows, cols, cols + qpad, nn.I8), s.matrix).run()
    got, gs = q.download(np.int8, (rows, cols + qpad)), s.get()[:, 0]
    fine = np.isfinite(x).all(axis=1)
    want, ws = U.quantised(x[fine])
    assert np.array_equal(gs[fine], ws) and np.isnan(gs[~fine]).all()
    assert np.array_equal(got[fine][:, :cols], want) and (got[~fine][:, :cols] == 0).all()
    to = min(-(-cols // 16) * 16, cols + qpad)
    assert (got[:, cols:to] == 0).all() and (got[:, to:] == 55).all()


I8_SIZES = [(1, 1, 1), (1, 64, 128), (3, 100, 7), (16, 512, 48), (17, 33, 64), (33, 130, 72), (64, 64, 64), (129, 500, 257), (300, 1000, 777),
            (2000, 64, 256), (40, 5000, 24)]


@pytest.mark.parametrize("rows,di,do", I8_SIZES)
@pytest.mark.parametrize("dtype,pad,shift", [(BF16, 0, 0), (F32, 3, 1), (F16, 16, 0)])
def test_i8_linear(rows, di, do, dtype, pad, shift):
    """The integer sum is exact; the scaled sum is off by the conversion and two products in single precision, and its type."""
    emit(f"i8 linear {rows} x {di}-{do} type {dtype} pad {pad}")
    g = np.random.default_rng(rows + di)
    x, w = U.rounded(g.standard_normal((rows, di)), dtype), g.integers(-127, 128, (do, di)).astype(np.int8)
    sw = np.exp(g.uniform(-7, -3, (do, 1))).astype(np.float32)
    hx, hw, hs, y, space = U.Held(x, dtype, pad, shift), U.Held(w, nn.I8, pad, shift), U.Held(sw, F32), U.Held(None, dtype, pad, shift, rows, do), U.Space()
    nn.I8Linear(hx.matrix, hw.matrix, hs.matrix, y.matrix, room=space).run()
    q, sx = U.quantised(x)
    want = (q.astype(np.float64) @ w.T.astype(np.float64)) * sx[:, None].astype(np.float64) * sw[:, 0].astype(np.float64)
    close("y", y.get(), want, (U.UNIT[dtype] + 3 * 2.0 ** -24) * abs(want) + 2.0 ** -25 * (dtype == F16))
    space.check()


@pytest.mark.parametrize("rows,di,f,do", [(1, 1, 1, 1), (1, 64, 128, 64), (5, 100, 60, 33), (33, 64, 256, 64), (70, 130, 200, 72), (129, 64, 256, 64),
                                          (1000, 96, 384, 40), (300, 32, 128, 96), (257, 128, 320, 128), (600, 520, 1000, 260)])
@pytest.mark.parametrize("dtype,name,pad,shift", [(BF16, "silu", 0, 0), (F32, "gelu", 3, 1), (F16, "relu", 16, 0)])
def test_i8_block(rows, di, f, do, dtype, name, pad, shift):
    """h is off by single precision's rounding, so a value of h that lies within it of the middle between two 8-bit steps may go
    to either: each such value may move y by one step of its row."""
    emit(f"i8 block {rows} x {di}-{f}-{do} type {dtype} {name} pad {pad}")
    g = np.random.default_rng(rows + f)
    x = U.rounded(g.standard_normal((rows, di)), dtype)
    ws = [g.integers(-127, 128, s).astype(np.int8) for s in ((f, di), (f, di), (do, f))]
    ss = [(np.exp(g.uniform(-0.5, 0.5, (n, 1))) / 73 / np.sqrt(k)).astype(np.float32) for n, k in ((f, di), (f, di), (do, f))]
    hx, y, space = U.Held(x, dtype, pad, shift), U.Held(None, dtype, pad, shift, rows, do), U.Space()
    hw, hs = [U.Held(w, nn.I8, pad, shift) for w in ws], [U.Held(s, F32) for s in ss]
    nn.I8FeedForward(hx.matrix, hw[0].matrix, hs[0].matrix, hw[1].matrix, hs[1].matrix, hw[2].matrix, hs[2].matrix, y.matrix, act=name,
                     room=space).run()
    dense = lambda q, s, w, sw: (q.astype(np.float64) @ w.T.astype(np.float64)) * s[:, None].astype(np.float64) * sw[:, 0].astype(np.float64)  # noqa: E731
    q, sx = U.quantised(x)
    gate, upv = dense(q, sx, ws[0], ss[0]), dense(q, sx, ws[1], ss[1])
    a, _ = U.act(name, gate)
    h = a * upv
    top = abs(h).max(axis=1, keepdims=True)
    step = top / 127
    off = (2.0 ** -20 * (abs(h) + abs(upv)) + 2.0 ** -20 * top)  # of h, and of the step times 127
    t = np.where(step > 0, h / np.where(step > 0, step, 1), 0)
    frac = abs(t - np.floor(t) - 0.5)
    unsure = frac <= off / np.where(step > 0, step, 1)
    want = (np.rint(t) @ ws[2].T.astype(np.float64)) * step * ss[2][:, 0].astype(np.float64)
    slack = (unsure @ abs(ws[2]).T.astype(np.float64)) * step * ss[2][:, 0]
    close("y", y.get(), want, (U.UNIT[dtype] + 2.0 ** -19) * abs(want) + slack + 2.0 ** -25 * (dtype == F16) + 1e-30)
    space.check()


def test_i8_rows_that_are_not_finite_or_zero():
    x = np.random.default_rng(1).standard_normal((50, 64))
    x[3], x[4, 5], x[6, 7] = 0, np.nan, -np.inf
    w = np.random.default_rng(2).integers(-127, 128, (96, 64)).astype(np.int8)
    d = np.random.default_rng(3).integers(-127, 128, (64, 96)).astype(np.int8)
    hx, hw, hd, s96, s64, space = U.Held(x, F32), U.Held(w, nn.I8), U.Held(d, nn.I8), U.Held(np.full((96, 1), 0.01), F32), U.Held(np.full((64, 1), 0.01), F32), U.Space()
    y, z = U.Held(None, F32, rows=50, cols=96), U.Held(None, F32, rows=50, cols=64)
    nn.I8Linear(hx.matrix, hw.matrix, s96.matrix, y.matrix, room=space).run()
    nn.I8FeedForward(hx.matrix, hw.matrix, s96.matrix, hw.matrix, s96.matrix, hd.matrix, s64.matrix, z.matrix, room=space).run()
    for got in (y.get(), z.get()):
        assert (got[3] == 0).all() and np.isnan(got[4]).all() and np.isnan(got[6]).all()
        assert np.isfinite(np.delete(got, (4, 6), axis=0)).all()
    space.check()
