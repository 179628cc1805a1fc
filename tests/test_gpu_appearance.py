"""The appearance example: the head learns the views' lighting from the rasterizer's gradients, and holds in 8 bits; and the C
ABI's handles give what the launchers give."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

from b2ctrain_amd import _native, nn
from tests import dense_util as U
from tests.gpu_harness import emit

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_appearance_head_learns_and_holds_in_8_bits():
    import appearance_head

    emit("appearance head: 2048 splats, 45 steps")
    start, full, eight = appearance_head.run(splats=2048, steps=45, say=emit)
    assert np.isfinite(full).all() and np.isfinite(eight).all()
    assert sum(full) < 0.7 * sum(start), (start, full)
    assert abs(sum(eight) - sum(full)) < 0.1 * sum(start), (full, eight)


def test_handles_give_what_the_launchers_give():
    L = _native.lib()
    for name, args in (("b2c_feed_forward", [C.c_void_p, C.POINTER(nn.FfnArgs), C.c_int, C.c_void_p]),
                       ("b2c_feed_forward_backward", [C.c_void_p, C.POINTER(nn.FfnGradArgs), C.c_void_p]),
                       ("b2c_i8_feed_forward", [C.c_void_p, C.POINTER(nn.I8FfnArgs), C.c_void_p])):
        getattr(L, name).argtypes = args
    L.b2c_dense_create.restype = C.c_void_p
    L.b2c_dense_destroy.argtypes = [C.c_void_p]
    d = L.b2c_dense_create()
    try:
        for rows, di, f in ((9, 64, 96), (300, 200, 330), (500, 64, 128)):
            emit(f"handle: {rows} x {di}-{f}")
            g = np.random.default_rng(rows)
            q = lambda *s: U.Held(g.standard_normal(s) * s[1] ** -0.5, nn.BF16)  # noqa: E731
            x, wg, wu, wd, dy = q(rows, di), q(f, di), q(f, di), q(di, f), q(rows, di)
            outs = []
            for handle in (False, True):
                space = U.Space()
                y, dx, dw = (U.Held(None, nn.BF16, rows=a, cols=b) for a, b in ((rows, di), (rows, di), (di, f)))
                ff = nn.FeedForward(x.matrix, wg.matrix, wu.matrix, wd.matrix, y.matrix, p=0.2, seed=3, train=True, room=space)
                ff.gradients(dy.matrix, dx=dx.matrix, dw_down=dw.matrix, room=space)
                if handle:
                    assert L.b2c_feed_forward(d, C.byref(ff.args), 1, None) == 0, L.b2c_last_error()
                    assert L.b2c_feed_forward_backward(d, C.byref(ff.grad), None) == 0, L.b2c_last_error()
                else:
                    ff.forward()
                    ff.backward()
                outs.append([y.get(), dx.get(), dw.get()])
            assert all(np.array_equal(a, b) for a, b in zip(*outs))
        ff.args.act = 17
        assert L.b2c_feed_forward(d, C.byref(ff.args), 1, None) != 0
        assert b"feed_forward: invalid arguments" in L.b2c_last_error()
        assert L.b2c_feed_forward(d, None, 1, None) != 0 and b"null" in L.b2c_last_error()
        big = nn.FfnGradArgs.from_buffer_copy(ff.grad)
        big.fwd.act, big.fwd.rows, big.fwd.d_in = 0, 1 << 20, 256
        assert L.b2c_feed_forward_backward(d, C.byref(big), None) != 0 and b"no forward pass" in L.b2c_last_error()
    finally:
        L.b2c_dense_destroy(d)
