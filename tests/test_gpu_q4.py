"""4-bit weights on the GPU: what quantising gives, to the bit, and products of it, against their restatement in 64 bits (more_util.py)."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests.gpu_harness import emit
from tests.test_gpu_dense import close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


class Bytes(U.Held):
    """Whole numbers of 8 or 32 bits, in a larger buffer like Held."""

    def __init__(self, x, np_type=np.uint8, pad=0, shift=0, rows=None, cols=None):
        from b2ctrain_amd import _native
        self.dtype = {np.uint8: nn.U8, np.int32: nn.I32}[np_type]
        self.rows, self.cols = (rows, cols) if x is None else x.shape
        self.ld, self.shift = self.cols + pad, shift
        flat = np.full(max(1, self.rows * self.ld + shift + 8), 113, np_type)
        if x is not None:
            self._window(flat)[:] = x
        self.before, self.np_type = flat, flat.dtype
        self.dev = _native.DeviceArray(flat)
        self.matrix = nn.Matrix(self.dev.ptr + shift * flat.itemsize, self.rows, self.cols, self.ld, self.dtype, keep=self.dev)

    def get(self):
        flat = self.dev.download(self.np_type, self.before.shape)
        got = self._window(flat).copy()
        self._window(flat)[:] = self._window(self.before)
        assert np.array_equal(flat, self.before), "values around the matrix changed"
        return got


def quantise(x, dtype, group, zeros, scale_dtype, pad=0, shift=0, values=True):
    rows, cols = x.shape
    n = V.groups(cols, group)
    emit(f"quantise {rows} x {cols} type {dtype} by {group} zeros {zeros} pad {pad} shift {shift}")
    h = U.Held(x, dtype, pad, shift)
    q, z = Bytes(None, pad=pad, shift=shift, rows=rows, cols=-(-cols // 2)), Bytes(None, pad=pad, rows=rows, cols=n)
    s, v = U.Held(None, scale_dtype, pad, shift, rows, n), U.Held(None, dtype, pad, shift, rows, cols)
    nn.QuantizeGroups(h.matrix, q.matrix, s.matrix, group, zero=z.matrix if zeros else None, values=v.matrix if values else None).run()
    code, stored, zero, exact = V.quantised4(x, group, zeros, scale_dtype)
    assert np.array_equal(s.get(), U.value(stored, scale_dtype), equal_nan=True)
    assert np.array_equal(q.get(), V.packed(code))
    if zeros:
        assert np.array_equal(z.get(), zero)
    if values:
        assert np.array_equal(v.get(), U.rounded(exact, dtype), equal_nan=True)
    return code, stored, zero


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (3, 31), (5, 32), (7, 33), (64, 64), (33, 100), (9, 255), (16, 256), (4, 257), (300, 1000), (2, 5001)])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype,scale_dtype", [(F32, BF16), (F16, F16), (BF16, BF16), (F32, F16)])
def test_quantise(rows, cols, group, zeros, dtype, scale_dtype):
    g = np.random.default_rng(rows + cols)
    quantise(U.rounded(g.standard_normal((rows, cols)) * np.exp(g.uniform(-3, 3, (rows, 1))), dtype), dtype, group, zeros, scale_dtype)


@pytest.mark.parametrize("pad,shift", [(1, 0), (3, 1), (8, 5)])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantise_strides(pad, shift, zeros):
    g = np.random.default_rng(1)
    for cols in (32, 45, 300):
        quantise(g.standard_normal((37, cols)).astype(np.float32), F32, 32, zeros, BF16, pad, shift, values=cols != 300)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale_dtype", [F16, BF16])
def test_quantise_groups_that_are_not_ordinary(zeros, scale_dtype):
    """Zeros, a single value, one sign, infinities, NaN, subnormals, scales beyond the type's range, ties."""
    g = np.random.default_rng(2)
    x = g.standard_normal((12, 96)).astype(np.float32)
    x[0] = 0
    x[1, :32] = -0.0
    x[2, :] = 0
    x[2, 40] = -3
    x[3] = abs(x[3])
    x[4] = -abs(x[4])
    x[5, 3], x[5, 40], x[5, 70] = np.inf, -np.inf, np.nan
    x[6] = np.float32(1e-45) * g.integers(0, 40, 96)
    x[7] *= np.float32(1e-30)
    x[8] *= np.float32(1e37)
    x[9] = 3.4e38 * np.sign(x[9])
    x[10] = g.integers(-14, 15, 96) * 0.5
    x[10, ::32], x[10, 1::32] = 7, -7
    x[11] = g.integers(0, 31, 96) * 0.5
    x[11, ::32], x[11, 1::32] = 15, 0
    quantise(x, F32, 32, zeros, scale_dtype)
    quantise(x, F32, 128, zeros, scale_dtype)


def linear(rows, k, n, group, zeros, dtype, pad=0, shift=0, x=None):
    emit(f"q4 linear {rows} x {k}-{n} by {group} zeros {zeros} type {dtype} pad {pad} shift {shift}")
    g = np.random.default_rng(rows + k + n)
    x = U.rounded(g.standard_normal((rows, k)), dtype) if x is None else x
    code = g.integers(0, 16, (n, k)).astype(np.uint8)
    m = V.groups(k, group)
    scale = U.rounded((0.5 + g.random((n, m))) / (4.6 * np.sqrt(k)), dtype)
    zero = g.integers(0, 16, (n, m)).astype(np.uint8) if zeros else np.full((n, m), 8, np.uint8)
    hx, hs, y, space = U.Held(x, dtype, pad, shift), U.Held(scale, dtype, pad, shift), U.Held(None, dtype, pad, shift, rows, n), U.Space()
    bits = V.packed(code)
    if k % 2:
        bits[:, -1] |= 0xA0  # what is behind an odd row's last column does not matter
    hw, hz = Bytes(bits, pad=pad, shift=shift), Bytes(zero, pad=pad, shift=shift)
    p = nn.Q4Linear(hx.matrix, hw.matrix, hs.matrix, y.matrix, group, zero=hz.matrix if zeros else None, room=space)
    p.run()
    got = y.get()
    close("y", got, *V.q4_linear(x, code, scale, zero, group, dtype, p.args.workspace_bytes == 0))
    p.run()
    assert np.array_equal(got, y.get())
    space.check()


@pytest.mark.parametrize("rows", [1, 3, 16, 17, 32, 33, 70, 200])
@pytest.mark.parametrize("k,n", [(1, 1), (33, 17), (64, 64), (127, 40), (128, 16), (300, 100), (1000, 333), (2050, 70), (4096, 48), (5000, 33)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (256, False)])
def test_linear(rows, k, n, group, zeros):
    linear(rows, k, n, group, zeros, BF16 if rows % 2 else F16)


@pytest.mark.parametrize("rows", [1, 9, 20, 40])
@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 1), (1, 3)])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (256, True)])
@pytest.mark.parametrize("k", [96, 515])
def test_linear_strides(rows, pad, shift, group, zeros, k):
    linear(rows, k, 50, group, zeros, BF16, pad, shift)


@pytest.mark.parametrize("rows", [1, 40])
def test_linear_of_rows_all_of_one_sign(rows):
    """Where the codes' base has the most to cancel."""
    g = np.random.default_rng(4)
    for dtype in (BF16, F16):
        linear(rows, 4096, 40, 128, False, dtype, x=U.rounded(1 + g.random((rows, 4096)), dtype))


@pytest.mark.parametrize("rows,k", [(1, 4096), (1, 500), (9, 512), (40, 512), (600, 300)])
def test_linear_of_subnormal_values(rows, k):
    """Which count like any others."""
    linear(rows, k, 40, 64, True, F16, x=np.random.default_rng(5).integers(-1000, 1001, (rows, k)) * 2.0 ** -24)


@pytest.mark.parametrize("rows,k,n", [(700, 600, 1100), (1300, 2048, 2048), (129, 4096, 520), (513, 4090, 4110)])
def test_linear_larger(rows, k, n):
    linear(rows, k, n, 128, True, BF16)


def test_no_rows():
    b, s = Bytes(np.zeros((4, 4), np.uint8)), U.Held(np.ones((4, 1)), BF16)
    none = nn.Matrix(s.matrix.ptr, 0, 8, 8, BF16)
    nn.Q4Linear(none, b.matrix, s.matrix, nn.Matrix(s.matrix.ptr, 0, 4, 4, BF16), 32).run()
    nn.QuantizeGroups(none, nn.Matrix(b.matrix.ptr, 0, 4, 4, nn.U8), nn.Matrix(s.matrix.ptr, 0, 1, 1, BF16), 32).run()
