"""Calls of the norms, 4-bit products and experts that differ from the usual ones in one thing: recorded and replayed, through a handle, on
two streams at once, rows so far apart that their places pass 32 bits."""
import ctypes as C

import numpy as np
import pytest

from b2ctrain_amd import _native, nn
from tests import dense_util as U
from tests import more_util as V
from tests.gpu_harness import emit
from tests.test_gpu_dense import Graph, close
from tests.test_gpu_dense_calls import Raw
from tests.test_gpu_q4 import Bytes

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


class Block:
    """Norm, experts, norm with gate and residual and its gradients, and a 4-bit head whose weights are made on the way."""

    def __init__(self, rows, d, f, e, k, seed):
        g = np.random.default_rng(seed)
        q = lambda *s, k=1.0: U.Held(g.standard_normal(s) * k, BF16)  # noqa: E731
        new = lambda r, c, t=BF16: U.Held(None, t, rows=r, cols=c)  # noqa: E731
        self.space = U.Space()
        x, self.wr, wg, wu, wd = q(rows, d), q(e, d), q(e * f, d, k=d ** -0.5), q(e * f, d, k=d ** -0.5), q(e * d, f, k=f ** -0.5)
        gate, w1, w2, dy, dn, head = q(1, d), q(1, d), q(1, d), q(rows, d), q(rows, d), U.Held(g.standard_normal((72, d)), F32)
        n = V.groups(d, 32)
        bits, scale, zero = Bytes(None, rows=72, cols=-(-d // 2)), new(72, n), Bytes(None, rows=72, cols=n)
        n1, y1, y2, n2, y3, dx, dr, dg = (new(r, c) for r, c in ((rows, d), (rows, d), (rows, d), (rows, d), (rows, 72), (rows, d), (rows, d), (1, d)))
        dw = [new(1, d, F32) for _ in range(2)]
        self.index = Bytes(None, np.int32, rows=rows, cols=k)
        self.open = nn.BlockNorm(residual=x.matrix, n=n1.matrix, w_pre=w1.matrix)
        self.experts = nn.Experts(n1.matrix, self.wr.matrix, wg.matrix, wu.matrix, wd.matrix, y1.matrix, k, index=self.index.matrix, room=self.space)
        self.close = nn.BlockNorm(x=y1.matrix, residual=x.matrix, gate=gate.matrix, gate_act="sigmoid", post=True, w_post=w1.matrix, w_pre=w2.matrix,
                                  y=y2.matrix, n=n2.matrix, kind="layer")
        self.close.gradients(dy=dy.matrix, dn=dn.matrix, dx=dx.matrix, dresidual=dr.matrix, dgate=dg.matrix, dw_post=dw[0].matrix,
                             dw_pre=dw[1].matrix, room=self.space)
        self.pack = nn.QuantizeGroups(head.matrix, bits.matrix, scale.matrix, 32, zero=zero.matrix)
        self.head = nn.Q4Linear(n2.matrix, bits.matrix, scale.matrix, y3.matrix, 32, zero=zero.matrix, room=self.space)
        self.out = [n1, y1, y2, n2, y3, dx, dr, dg, *dw, self.index]
        self.keep = [x, wg, wu, wd, gate, w1, w2, dy, dn, head, bits, scale, zero]

    def run(self, stream):
        self.open.forward(stream)
        self.experts.run(stream)
        self.close.forward(stream)
        self.close.backward(stream)
        self.pack.run(stream)
        self.head.run(stream)

    def results(self):
        return [o.get() for o in self.out]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("rows,d,f,e,k", [(1, 96, 80, 8, 2), (1, 40, 24, 300, 3), (30, 96, 80, 8, 2), (300, 130, 40, 4, 4), (700, 64, 48, 5, 1)])
def test_recorded_calls_replay(rows, d, f, e, k):
    """From a recorded graph, between eager passes of another block into the same outputs."""
    emit(f"graph {rows} x {d}-{f}, {k} of {e}")
    a, b = Block(rows, d, f, e, k, 1), Block(rows, d, f, e, k, 2)
    L = _native.lib()
    ctx = L.b2c_ctx_create()
    try:
        s = L.b2c_ctx_stream(ctx)
        a.run(s)
        assert L.b2c_ctx_synchronize(ctx) == 0
        want = a.results()
        graph = Graph(s, a.run)
        for i in range(3):
            for p, q in ((a.open, b.open), (a.close, b.close)):  # the other block's values in this one's outputs
                q.args.y, q.args.n = p.args.y, p.args.n
            b.experts.args.y, b.head.args.y = a.experts.args.y, a.head.args.y
            b.run(s)
            assert L.b2c_ctx_synchronize(ctx) == 0
            assert not any(np.array_equal(x, y) for x, y in zip(want[:5], a.results()[:5]))
            graph.replay()
            assert same(want, a.results()), i
        graph.close()
    finally:
        L.b2c_ctx_destroy(ctx)
    a.space.check()


def test_two_blocks_on_two_streams_at_once():
    blocks = [Block(200, 256, 128, 16, 4, seed) for seed in (3, 4)]
    want = []
    for b in blocks:
        b.run(0)
        want.append(b.results())
    L = _native.lib()
    ctx = [L.b2c_ctx_create() for _ in blocks]
    try:
        for _ in range(5):
            for b, c in zip(blocks, ctx):
                b.run(L.b2c_ctx_stream(c))
        assert all(L.b2c_ctx_synchronize(c) == 0 for c in ctx)
        assert all(same(w, b.results()) for w, b in zip(want, blocks))
    finally:
        for c in ctx:
            L.b2c_ctx_destroy(c)


def test_handles_give_what_the_launchers_give():
    L, p = _native.lib(), C.c_void_p
    names = {"b2c_block_norm": nn.BlockNormArgs, "b2c_block_norm_backward": nn.BlockNormGradArgs, "b2c_quantize4": nn.Quantize4Args,
             "b2c_q4_linear": nn.Q4LinearArgs, "b2c_experts": nn.ExpertsArgs}
    for name, args in names.items():
        getattr(L, name).argtypes = [C.POINTER(args), p] if name in ("b2c_block_norm", "b2c_quantize4") else [p, C.POINTER(args), p]
    L.b2c_dense_create.restype, L.b2c_dense_destroy.argtypes = p, [p]
    d = L.b2c_dense_create()
    try:
        for rows in (1, 40, 700):  # one handle for calls whose workspaces differ
            b = Block(rows, 96, 80, 8, 2, rows)
            b.run(0)
            want = b.results()
            for call in (lambda: L.b2c_block_norm(C.byref(b.open.args), None), lambda: L.b2c_experts(d, C.byref(b.experts.args), None),
                         lambda: L.b2c_block_norm(C.byref(b.close.args), None), lambda: L.b2c_block_norm_backward(d, C.byref(b.close.grad), None),
                         lambda: L.b2c_quantize4(C.byref(b.pack.args), None), lambda: L.b2c_q4_linear(d, C.byref(b.head.args), None)):
                assert call() == 0, L.b2c_last_error()
            assert same(want, b.results())
    finally:
        L.b2c_dense_destroy(d)


# ---- rows far apart ----------------------------------------------------------------------------------------

class Far:
    """rows x cols 16-bit (or 8-bit) values `ld` apart, of which some are written."""

    def __init__(self, rows, cols, ld, dtype=F16):
        self.raw, self.cols, self.ld, self.dtype = Raw((rows - 1) * ld + cols, np.uint8 if dtype == nn.U8 else np.float16), cols, ld, dtype
        self.matrix = nn.Matrix(self.raw.ptr.value, rows, cols, ld, dtype)

    def write(self, row, v):
        self.raw.write(row * self.ld, v)

    def read(self, row):
        return self.raw.read(row * self.ld, self.cols).astype(np.float64)

    def free(self):
        self.raw.free()


def test_block_norm_of_rows_far_apart():
    rows, d, ld = 1100, 48, 1 << 22  # 9 GiB each
    emit(f"block norm {rows} x {d}, rows {ld} apart")
    g = np.random.default_rng(1)
    v = {k: U.rounded(g.standard_normal((rows, d)), F16) for k in ("x", "r", "dy", "dn")}
    far = {k: Far(rows, d, ld) for k in ("x", "r", "y", "dx")}
    try:
        for k in ("x", "r"):
            for i in range(rows):
                far[k].write(i, v[k][i])
        h = {k: U.Held(v[k], F16) for k in ("dy", "dn")}
        n = U.Held(None, F16, rows=rows, cols=d)
        p = nn.BlockNorm(x=far["x"].matrix, residual=far["r"].matrix, y=far["y"].matrix, n=n.matrix, post=True)
        p.gradients(dy=h["dy"].matrix, dn=h["dn"].matrix, dx=far["dx"].matrix, room=U.Space())
        p.forward()
        p.backward()
        want = V.block_norm(F16, F16, x=v["x"], r=v["r"], post=True, dy=v["dy"], dn=v["dn"])
        close("n", n.get(), *want["n"])
        for i in (0, 511, 512, 1099):
            close(f"y of row {i}", far["y"].read(i), want["y"][0][i], want["y"][1][i])
            close(f"dx of row {i}", far["dx"].read(i), want["dx"][0][i], want["dx"][1][i])
    finally:
        for f in far.values():
            f.free()


@pytest.mark.parametrize("rows", [1, 9, 40, 600])
@pytest.mark.parametrize("k", [100, 2048])
def test_q4_linear_of_rows_far_apart(rows, k):
    n, ld, group = 264, 1 << 25, 64  # 8.25 GiB of codes and twice that of scales
    emit(f"q4 linear {rows} x {k}-{n}, rows {ld} apart")
    g = np.random.default_rng(k)
    m = V.groups(k, group)
    x = U.rounded(g.standard_normal((rows, k)), F16)
    code, scale = g.integers(0, 16, (n, k)).astype(np.uint8), U.rounded(0.05 + 0.05 * g.random((n, m)), F16)
    w, s = Far(n, k // 2, ld, nn.U8), Far(n, m, ld)
    try:
        for i, bits in enumerate(V.packed(code)):
            w.write(i, bits)
            s.write(i, scale[i])
        hx, y, space = U.Held(x, F16), U.Held(None, F16, rows=rows, cols=n), U.Space()
        p = nn.Q4Linear(hx.matrix, w.matrix, s.matrix, y.matrix, group, room=space)
        p.run()
        close("y", y.get(), *V.q4_linear(x, code, scale, np.full((n, m), 8), group, F16, p.args.workspace_bytes == 0))
    finally:
        w.free()
        s.free()


@pytest.mark.parametrize("rows", [1, 20])
def test_experts_of_rows_far_apart(rows):
    e, d, f, o, ld = 9, 24, 18, 20, 1 << 25  # 9 x 18 rows of 64 MiB
    emit(f"experts {rows} x {d}-{f}-{o}, rows {ld} apart")
    g = np.random.default_rng(2)
    q = lambda *s: U.rounded(g.standard_normal(s) * 0.3, F16)  # noqa: E731
    v = dict(x=q(rows, d), wr=q(e, d), wg=q(e * f, d), wu=q(e * f, d), wd=q(e * o, f))
    far = dict(wg=Far(e * f, d, ld), wu=Far(e * f, d, ld), wd=Far(e * o, f, ld))
    try:
        for k, m in far.items():
            for i in range(len(v[k])):
                m.write(i, v[k][i])
        hx, hr, y = U.Held(v["x"], F16), U.Held(v["wr"], F16), U.Held(None, F16, rows=rows, cols=o)
        nn.Experts(hx.matrix, hr.matrix, far["wg"].matrix, far["wu"].matrix, far["wd"].matrix, y.matrix, 4, room=U.Space()).run()
        _, _, want, bound = V.experts(v["x"], v["wr"], v["wg"], v["wu"], v["wd"], 4, "silu", F16)
        close("y", y.get(), want, bound)
    finally:
        for m in far.values():
            m.free()


def test_quantise_of_more_rows_than_a_launch_has_threads():
    """32 columns are four threads a row: 2^30 rows and four lanes each."""
    rows, n = (1 << 30) - 5, 500
    emit(f"quantise {rows} x 2, 7 GB")
    x, q, s = Raw(rows * 2, np.float16), Raw(rows, np.uint8), Raw(rows, np.float16)
    try:
        parts = {first: np.random.default_rng(first % 97).standard_normal((n, 2)).astype(np.float16) for first in (0, (1 << 29) - 250, rows - n)}
        for first, v in parts.items():
            x.write(first * 2, v)
        nn.QuantizeGroups(nn.Matrix(x.ptr.value, rows, 2, 2, F16), nn.Matrix(q.ptr.value, rows, 1, 1, nn.U8), nn.Matrix(s.ptr.value, rows, 1, 1, F16), 32).run()
        for first, v in parts.items():
            code, scale, _, _ = V.quantised4(v.astype(np.float32), 32, False, F16)
            assert np.array_equal(q.read(first, n), V.packed(code)[:, 0]) and np.array_equal(s.read(first, n), scale[:, 0]), first
    finally:
        for m in (x, q, s):
            m.free()
