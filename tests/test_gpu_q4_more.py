"""Products with 4-bit weights where the size, the range or the precision is at its limit."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests import precision as P
from tests.gpu_harness import emit
from tests.test_gpu_dense import close
from tests.test_gpu_dense_calls import Raw
from tests.test_gpu_q4 import Bytes, linear

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def test_more_than_four_million_workgroups_of_weights():
    """Weights whose unpacking takes just more workgroups than one dimension of a launch holds, so that a launch has some without work,
    while x is read in place and there is nothing to copy: 17 GB of codes, 69 GB of workspace. Of the weights' rows some are written, from
    all over; the others hold what the memory holds."""
    rows, k, n, group = 513, 1 << 20, 32776, 256
    blocks = n * (k // 8) // 1024
    assert blocks > 1 << 22 and rows > 512
    emit(f"q4 linear {rows} x {k}-{n}, {blocks} workgroups")
    g = np.random.default_rng(1)
    x = ((g.integers(0, 1 << 16, (rows, k), dtype=np.uint16) & 0x83FF) | 0x3800).view(np.float16)  # 0.5 to 1, of either sign
    at = np.r_[0:3, 4096, 8191, 16388, 21001:21003, n - 9:n]
    code, scale = g.integers(0, 16, (len(at), k), dtype=np.uint8), g.uniform(0.5, 1, (len(at), k // group)).astype(np.float16) / 4096
    h = np.float16
    hx, q, s, y, space = Raw(rows * k, h), Raw(n * (k // 2), np.uint8), Raw(n * (k // group), h), Raw(rows * n, h), []

    def room(size):
        space.append(Raw(size, np.uint8))
        return nn.Matrix(space[-1].ptr.value, 1, size, size, nn.U8)

    try:
        hx.write(0, x.reshape(-1))
        for i, bits, v in zip(at, V.packed(code), scale):
            q.write(int(i) * (k // 2), bits)
            s.write(int(i) * (k // group), v)
        matrix = lambda raw, r, c, t: nn.Matrix(raw.ptr.value, r, c, c, t)  # noqa: E731
        p = nn.Q4Linear(matrix(hx, rows, k, F16), matrix(q, n, k // 2, nn.U8), matrix(s, n, k // group, F16), matrix(y, rows, n, F16), group, room=room)
        assert p.args.workspace_bytes > 2 * n * k
        p.run()
        want, size = np.zeros((rows, len(at))), np.zeros((rows, len(at)))
        for first in range(0, k, 1 << 16):
            part = slice(first, first + (1 << 16))
            w = (code[:, part] - 8.0) * np.repeat(scale[:, first // group:(first + (1 << 16)) // group].astype(np.float64), group, axis=1)
            v = x[:, part].astype(np.float64)
            want += v @ w.T
            size += np.square(v) @ np.square(w).T
        # y is rounded, and sums of products of either sign in single precision are off by some of the sum of squares' root, 2^-24 sqrt k of it if
        # their roundings know nothing of each other
        got = np.stack([y.read(m * n, n)[at] for m in range(rows)]).astype(np.float64)
        close("y", got, want, 2.0 ** -11 * abs(want) + 2.0 ** -12 * np.sqrt(size) + 2.0 ** -25)
    finally:
        for raw in (hx, q, s, y, *space):
            raw.free()


@pytest.mark.parametrize("rows", [1, 5, 17, 32, 33, 64, 200, 520, 700])
@pytest.mark.parametrize("k,n", [(4096, 600), (2050, 1040), (515, 900), (128, 2048)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (256, False)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_products_are_as_exact_as_their_outputs(rows, k, n, group, zeros, dtype):
    """Whatever the number of rows: weights of whole numbers and scales are nowhere rounded to 16 bits."""
    emit(f"q4 linear {rows} x {k}-{n} by {group} zeros {zeros} type {dtype}")
    x, code, scale, zero, w = P.weights4(rows, k, n, group, zeros, dtype)
    hx, hs, hw, hz, y = U.Held(x, dtype), U.Held(scale, dtype), Bytes(V.packed(code)), Bytes(zero), U.Held(None, dtype, rows=rows, cols=n)
    space = U.Space()
    nn.Q4Linear(hx.matrix, hw.matrix, hs.matrix, y.matrix, group, zero=hz.matrix if zeros else None, room=space).run()
    assert P.excess(y.get(), x @ w.T, dtype) < (P.MOST if rows * n > 2000 else 1.2)
    space.check()


def product(x, dtype, group, zeros, n=70, size=1.0, seed=3):
    """y of x and weights of about `size` each, those weights' codes, scales and zero points, and whether x goes by codes."""
    g = np.random.default_rng(seed)
    rows, k = x.shape
    code, m = g.integers(0, 16, (n, k)).astype(np.uint8), V.groups(k, group)
    scale = U.rounded((0.5 + g.random((n, m))) * size, dtype)
    zero = g.integers(0, 16, (n, m)).astype(np.uint8) if zeros else np.full((n, m), 8, np.uint8)
    hx, hs, hw, hz, y = U.Held(x, dtype), U.Held(scale, dtype), Bytes(V.packed(code)), Bytes(zero), U.Held(None, dtype, rows=rows, cols=n)
    p = nn.Q4Linear(hx.matrix, hw.matrix, hs.matrix, y.matrix, group, zero=hz.matrix if zeros else None, room=U.Space())
    p.run()
    return y.get(), code, scale, zero, p.args.workspace_bytes == 0


@pytest.mark.parametrize("rows", [1, 5, 20, 40, 600])
@pytest.mark.parametrize("k", [40, 300, 2048, 4100])
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False), (256, True)])
@pytest.mark.parametrize("dtype,largest", [(BF16, 3.3e38), (F16, 65504.0)])
def test_the_largest_values(rows, k, group, zeros, dtype, largest):
    """Any number of x, where y is one, whatever the number of rows."""
    emit(f"q4 linear {rows} x {k}, values of {largest}")
    g = np.random.default_rng(rows + k)
    x = U.rounded(g.uniform(0.5, 1, (rows, k)) * np.where(g.random((rows, k)) < 0.5, -largest, largest), dtype)
    x[rows // 2] = abs(x[rows // 2])  # and of one sign
    y, code, scale, zero, few = product(x, dtype, group, zeros, size=2.0 ** -10 / k)
    close("y", y, *V.q4_linear(x, code, scale, zero, group, dtype, few))


@pytest.mark.parametrize("rows", [1, 5, 20, 40, 600])
@pytest.mark.parametrize("k", [40, 300, 2048, 4100])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_with_infinities_or_nan(rows, k, dtype):
    """No number of such a row of y, and the others as without."""
    emit(f"q4 linear {rows} x {k}, not finite")
    g = np.random.default_rng(rows + k)
    x = U.rounded(g.standard_normal((rows, k)), dtype)
    clean, code, scale, zero, few = product(x, dtype, 64, True, size=k ** -0.5)
    close("y", clean, *V.q4_linear(x, code, scale, zero, 64, dtype, few))
    bad, at = sorted({0, rows // 2}), int(g.integers(k))
    for value in (np.inf, -np.inf, np.nan):
        for m in bad:
            x[m, at] = value
        y = product(x, dtype, 64, True, size=k ** -0.5)[0]
        assert not np.isfinite(y[bad]).any()
        others = np.setdiff1d(np.arange(rows), bad)
        assert np.array_equal(y[others], clean[others])


@pytest.mark.parametrize("rows", [1, 5, 20, 40, 600])
@pytest.mark.parametrize("k", [300, 4100])
def test_the_smallest_normal_values(rows, k):
    """bfloat16 down to 2^-126, by weights that make y of it about 1."""
    g = np.random.default_rng(rows + k)
    x = U.rounded(g.standard_normal((rows, k)) * 2.0 ** -123, BF16)
    x[abs(x) < 2.0 ** -126] = 2.0 ** -126
    y, code, scale, zero, few = product(x, BF16, 64, True, size=2.0 ** 110)
    close("y", y, *V.q4_linear(x, code, scale, zero, 64, BF16, few))


@pytest.mark.parametrize("k,n", [(1, 1), (7, 3), (33, 17), (64, 65), (97, 129), (515, 50), (1000, 333), (4128, 200)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (5, 1)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (256, False)])
def test_many_rows_of_every_width(k, n, pad, shift, group, zeros):
    """By tiles: steps that end inside a group, groups that end inside a step, parts of k, x in place and copied."""
    for dtype in (BF16, F16):
        linear(513 + n, k, n, group, zeros, dtype, pad, shift)
