"""The norms' sums over rows, and their ranges."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests.gpu_harness import emit
from tests.test_gpu_block_norm import check
from tests.test_gpu_dense import close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def whole_sums(rows, d, per, dtype, pad=0, accumulate=False):
    """Rows of 1 and -1, which are their own norms, a gate of 1 and -1, and whole gradients whose part along the row is zero: every term of the
    sums over rows is a whole number of 0 to 9, and so is every sum. Where the columns times their inverse are 1 in single precision the norms
    are exact, and so then are the sums; else a norm is off by up to 4 units in the last place, and each sum by no more than that, and a unit
    for each of 200 additions, of its terms' magnitudes: less than the smallest term of one row, so that none can be missing or counted
    twice."""
    emit(f"block norm {rows} x {d} type {dtype} per {per} pad {pad}: sums of whole numbers")
    g = np.random.default_rng(rows + d + per)
    signs = lambda *s: np.where(g.random(s) < 0.5, -1.0, 1.0)  # noqa: E731
    ints = lambda: signs(rows, d) * g.integers(1, 4, (rows, d))  # noqa: E731
    u, gate = signs(rows, d), signs(-(-rows // per), d)
    wide = gate[np.arange(rows) // per]
    v = u * wide  # y, and its norm
    dy, dn = ints() * 2, ints()  # their sum is no zero
    even = d // 2 * 2
    dn[:, 1:even:2] = -dn[:, 0:even:2] * v[:, 0:even:2] * v[:, 1:even:2]
    dn[:, even:] = 0
    start = g.integers(-50, 50, (2, d)).astype(np.float64) * accumulate
    h = {k: U.Held(a, dtype, pad) for k, a in (("x", u), ("gate", gate), ("dy", dy), ("dn", dn))}
    n, dg, one = U.Held(None, dtype, pad, 0, rows, d), U.Held(None, dtype, pad, 0, len(gate), d), U.Held(np.ones((1, d)), dtype)
    dw = [U.Held(start[i:i + 1], F32) for i in range(2)]
    p = nn.BlockNorm(x=h["x"].matrix, n=n.matrix, gate=h["gate"].matrix, rows_per_gate=per, post=True, w_post=one.matrix, w_pre=one.matrix, eps=0.0)
    space = U.Space()
    p.gradients(dy=h["dy"].matrix, dn=h["dn"].matrix, dgate=dg.matrix, dw_post=dw[0].matrix, dw_pre=dw[1].matrix, accumulate=accumulate, room=space)
    p.forward()
    p.backward()
    space.check()
    exact = np.float32(d) * (np.float32(1) / np.float32(d)) == 1
    assert not exact or np.array_equal(n.get(), v)
    terms = {"dw_post": (wide * (dy + dn) * u, dw[0].get()[0] - start[0]), "dw_pre": (dn * v, dw[1].get()[0] - start[1]),
             "dgate": ((dy + dn) * u, dg.get())}
    for k, (t, got) in terms.items():
        if k == "dgate":
            first = np.arange(0, rows, per)
            want, size = np.add.reduceat(t, first, axis=0), np.add.reduceat(abs(t), first, axis=0)
        else:
            want, size = t.sum(axis=0), abs(t).sum(axis=0)
        off = 0 * size if exact else (4 + 200) * 2.0 ** -24 * (size + abs(start).max())
        assert (off < 1).all()
        if k == "dgate":
            off = off + (U.UNIT[dtype] * (abs(want) + off) if dtype != F32 or not exact else 0)
        close(k, got, want, off)


# More rows than the workgroups have teams together: 32 teams of 8 lanes in each of 1024, 16 of 16, ... one of 256, 512 and 1024 lanes.
@pytest.mark.parametrize("rows,d", [(80001, 3), (70000, 16), (70001, 32), (40001, 64), (30000, 45), (20001, 128), (9001, 256), (5003, 1000),
                                    (5000, 1024), (2500, 2048), (1300, 2049), (1100, 4096), (700, 5001), (1100, 8192), (600, 9001),
                                    (700, 16384), (600, 16383), (9001, 47), (600, 8437)])
@pytest.mark.parametrize("per", ["all", "some"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sums_over_many_rows(rows, d, per, dtype):
    whole_sums(rows, d, rows if per == "all" else 61, dtype)


@pytest.mark.parametrize("rows,d,per", [(40001, 64, 1), (40000, 64, 2), (40001, 64, 3), (40001, 64, 16), (40001, 64, 20000), (5000, 1024, 2500),
                                        (700, 8192, 1), (700, 8192, 350), (700, 16384, 2), (600, 9001, 299)])
def test_sums_by_gate_rows(rows, d, per):
    for dtype in (BF16, F32):
        whole_sums(rows, d, per, dtype)


def test_sums_added_to_what_is_there():
    for rows, d in ((40001, 64), (5003, 1000), (700, 8192)):
        whole_sums(rows, d, rows, F32, pad=5, accumulate=True)


@pytest.mark.parametrize("d,dtype", [(9001, BF16), (16383, F16), (5001, F32), (9001, F32), (16383, F32)])
def test_wide_rows_that_end_inside_a_piece(d, dtype):
    """Rows of two and four pieces a thread."""
    check(19, d, dtype, kind="layer")
    check(300, d, dtype, F32, per=7, act="sigmoid")


@pytest.mark.parametrize("d,dtype", [(8192, BF16), (16384, BF16), (8192, F32), (16384, F32)])
@pytest.mark.parametrize("per", [0, 13, 350])
def test_more_wide_rows_than_workgroups(d, dtype, per):
    check(700, d, dtype, F32, per=per, act="sigmoid" if per else "none")
