"""The norms' sums over rows, and their ranges."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests import precision as P
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


def norms_of(u, dtype, kind, eps, gate=None):
    """norm(u) and its gradient of dn, on the GPU and in 64 bits."""
    rows, d = u.shape
    g = np.random.default_rng(rows + d)
    dn = U.rounded(g.standard_normal((rows, d)), dtype)
    hx, hn, n, dx = U.Held(u, dtype), U.Held(dn, dtype), U.Held(None, dtype, rows=rows, cols=d), U.Held(None, dtype, rows=rows, cols=d)
    p = nn.BlockNorm(residual=hx.matrix, n=n.matrix, kind=kind, eps=eps)
    p.gradients(dn=hn.matrix, dresidual=dx.matrix, room=U.Space())
    p.forward()
    p.backward()
    mean = lambda v: v.mean(axis=1, keepdims=True)  # noqa: E731
    c = u - mean(u) if kind == "layer" else u
    size = 1 / np.sqrt(mean(c * c) + float(np.float32(eps)))
    v = c * size
    back = dn - v * mean(dn * v) - (mean(dn) if kind == "layer" else 0)
    return (n.get(), v), (dx.get(), size * back, size * (abs(dn) + abs(v) + 1))


@pytest.mark.parametrize("d", [3, 33, 64, 200, 520, 1500, 4096, 5001, 16384])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("size", [1e17, 1.7e19, 3e19, 1e25, 3e37])
def test_rows_whose_squares_pass_the_range(d, dtype, kind, size):
    """A finite row has its norm, whatever its size, and the gradients that go with it."""
    emit(f"norm of rows of {d} values of about {size}, type {dtype} {kind}")
    u = U.rounded(np.random.default_rng(d).standard_normal((40, d)) * size * np.logspace(-0.4, 0.4, 40)[:, None], dtype)
    u[7] = U.rounded(np.random.default_rng(1).standard_normal(d), dtype)  # and an ordinary row among them
    u[9], u[9, d // 2] = 0, u[10, 0]
    (n, v), (dx, back, terms) = norms_of(u, dtype, kind, 1e-6)
    # statistics to 2^-18 of themselves at most, at the widths here, outputs rounded once; a layer norm's differences are of rounded means
    close("n", n, v, U.UNIT[dtype] * abs(v) + 2.0 ** -18 * (abs(v) + 1))
    close("dresidual", dx, back, U.UNIT[dtype] * abs(back) + 2.0 ** -16 * terms + 2.0 ** -133)


@pytest.mark.parametrize("d", [3, 64, 520, 4096, 5001])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e-12, 1e-19, 1e-24, 1e-36])
def test_small_rows_without_eps(d, dtype, size):
    emit(f"norm of rows of {d} values of about {size}, type {dtype}")
    u = U.rounded(np.random.default_rng(d).standard_normal((40, d)) * size, dtype)
    (n, v), _ = norms_of(u, dtype, "rms", 0.0)
    close("n", n, v, U.UNIT[dtype] * abs(v) + 2.0 ** -18 * (abs(v) + 1))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("per", [1, 64])
def test_sigmoids_far_from_zero(dtype, per):
    """A gate of 1 / (1 + e^-g) and its slope keep their relative precision on both sides, down to the type's smallest normal values."""
    rows, d = 64, 200
    g = np.random.default_rng(per)
    most = {BF16: 80, F16: 9, F32: 80}[dtype]
    gate, x, dy = (U.rounded(v, dtype) for v in (g.uniform(-most, most, (rows // per, d)), g.uniform(1, 2, (rows, d)), g.uniform(1, 2, (rows, d))))
    h = {k: U.Held(v, dtype) for k, v in (("x", x), ("gate", gate), ("dy", dy))}
    y, dg = U.Held(None, dtype, rows=rows, cols=d), U.Held(None, dtype, rows=rows // per, cols=d)
    p = nn.BlockNorm(x=h["x"].matrix, gate=h["gate"].matrix, rows_per_gate=per, gate_act="sigmoid", y=y.matrix, scale=0.5)
    p.gradients(dy=h["dy"].matrix, dgate=dg.matrix, room=U.Space())
    p.forward()
    p.backward()
    raw = np.repeat(gate, per, axis=0)
    s, rest = 1 / (1 + np.exp(-raw)), 1 / (1 + np.exp(raw))
    # In single precision: an exponential, a sum, a quotient, each within two units, and up to four products; sums of 64 rows six or more
    # additions of terms of one sign. In 16 bits the exponential's argument is rounded too, and the quotient is an approximation.
    off = (32 + (2 * abs(raw) + 32) * (dtype != F32)) * 2.0 ** -24 * np.ones_like(raw)
    want = 0.5 * s * x
    close("y", y.get(), want, (U.UNIT[dtype] + off) * want * 1.01)
    terms = 0.5 * dy * x * s * rest
    want = terms.reshape(-1, per, d).sum(axis=1)
    close("dgate", dg.get(), want, (U.UNIT[dtype] + (off + 64 * 2.0 ** -24).max(axis=0)) * want * 1.01 + 2.0 ** -25 * (dtype == F16))


@pytest.mark.parametrize("d", [3, 8, 24, 45, 64, 200, 600, 1000, 2048, 2500, 5000, 5001, 9000, 16384])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("post", [False, True])
def test_an_infinite_gate_makes_a_row_infinitely_large(d, dtype, post):
    """As an infinity in x does: the other values of its norm are zeros, in every width."""
    rows = 9
    g = np.random.default_rng(d)
    x, gate = (U.rounded(g.uniform(1, 2, (rows, d)), dtype) for _ in range(2))
    at = {2: 0, 5: d // 2, 7: d - 1}
    clean = gate.copy()
    for m, c in at.items():
        gate[m, c] = np.inf
    y, n = U.Held(None, dtype, rows=rows, cols=d), U.Held(None, dtype, rows=rows, cols=d)
    for v in (clean, gate):
        nn.BlockNorm(x=U.Held(x, dtype).matrix, gate=U.Held(v, dtype).matrix, rows_per_gate=1, post=post, y=y.matrix, n=n.matrix).forward()
        if v is clean:
            want = y.get(), n.get()
    y, n = y.get(), n.get()
    for m, c in at.items():
        others = np.arange(d) != c
        assert y[m, c] == np.inf and np.array_equal(y[m, others], want[0][m, others])
        assert np.isnan(n[m, c]) and not n[m, others].any()
    rest = [m for m in range(rows) if m not in at]
    assert np.array_equal(y[rest], want[0][rest]) and np.array_equal(n[rest], want[1][rest])


def test_batches_of_no_rows():
    """An empty batch's matrices have no address; the weights' gradients of it are zeros, or stay as they are."""
    none = lambda: nn.Matrix(0, 0, 40, 40, BF16)  # noqa: E731
    w, dw = U.Held(np.ones((1, 40)), F32), [U.Held(np.ones((1, 40)), F32) for _ in range(2)]
    p = nn.BlockNorm(x=none(), residual=none(), y=none(), n=none(), post=True, w_post=w.matrix, w_pre=w.matrix)
    p.forward()
    for accumulate in (True, False):
        p.gradients(dy=none(), dn=none(), dx=none(), dresidual=none(), dw_post=dw[0].matrix, dw_pre=dw[1].matrix, accumulate=accumulate)
        p.backward()
        assert all(np.array_equal(v.get(), np.full((1, 40), float(accumulate))) for v in dw)


@pytest.mark.parametrize("rows,d,per", [(1037, 1000, 61), (300, 4096, 0), (5000, 300, 5000), (700, 8192, 350)])
def test_sums_over_rows_are_as_exact_as_their_terms(rows, d, per):
    """In single precision. A term has five roundings or so, each 2^-24 / sqrt 3 on the average, and the sum's own is a sixth: 8.4e-8 of it, where
    terms have either sign. To add a thousand workgroups' sums in single precision would bring another 1.4e-7."""
    emit(f"block norm {rows} x {d} per {per}: precision of the sums")
    g = np.random.default_rng(rows)
    q = lambda k, n=rows, add=0.0: U.rounded(g.standard_normal((n, d)) * k + add, F32)  # noqa: E731
    x, r, dy, dn, w_post, w_pre = q(0.5), q(2.0), q(0.1), q(0.1), q(0.2, 1, 1.0), q(0.2, 1, 1.0)
    gate = q(1.0, -(-rows // per)) if per else None
    h = [U.Held(v, F32) for v in (x, r, dy, dn, w_post, w_pre)]
    n, dw = U.Held(None, F32, rows=rows, cols=d), [U.Held(None, F32, rows=1, cols=d) for _ in range(2)]
    dg = U.Held(None, F32, rows=len(gate), cols=d) if per else None
    p = nn.BlockNorm(x=h[0].matrix, residual=h[1].matrix, n=n.matrix, gate=U.Held(gate, F32).matrix if per else None, rows_per_gate=per or None,
                     post=True, w_post=h[4].matrix, w_pre=h[5].matrix, scale=0.5)
    p.gradients(dy=h[2].matrix, dn=h[3].matrix, dgate=dg.matrix if per else None, dw_post=dw[0].matrix, dw_pre=dw[1].matrix, room=U.Space())
    p.backward()
    want = V.block_norm(F32, F32, x=x, r=r, gate=gate, per=per or 1, post=True, w_post=w_post[0], w_pre=w_pre[0], scale=0.5, dy=dy, dn=dn)
    for k, got in (("dw_post", dw[0].get()[0]), ("dw_pre", dw[1].get()[0]), ("dgate", dg.get() if per else None)):
        if got is not None:
            assert P.rms(got - want[k][0]) / P.rms(want[k][0]) < 1.25e-7, k
