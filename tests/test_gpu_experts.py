"""A mixture of experts for a few tokens against its restatement in 64 bits (more_util.py), and the operators between, in and after a block
run together."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests.gpu_harness import emit
from tests.test_gpu_dense import close
from tests.test_gpu_q4 import Bytes

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def make(rows, d, f, o, e, dtype, seed=0):
    g = np.random.default_rng(seed + rows + d + f + e)
    q = lambda *s, k=1.0: U.rounded(g.standard_normal(s) * k, dtype)  # noqa: E731
    return dict(x=q(rows, d), wr=q(e, d, k=2 * d ** -0.5), wg=q(e * f, d, k=d ** -0.5), wu=q(e * f, d, k=d ** -0.5),
                wd=q(e * o, f, k=f ** -0.5), r=q(rows, o))


def check(rows, d, f, o, e, k, dtype, name="silu", normalize=True, residual=False, pad=0, shift=0, values=None, in_place=False):
    emit(f"experts {rows} x {d}-{f}-{o}, {k} of {e}, type {dtype} {name} pad {pad} shift {shift}")
    v = make(rows, d, f, o, e, dtype)
    if values:
        v.update({n: U.rounded(a, dtype) for n, a in values(v).items()})  # what the device holds
    h = {n: U.Held(a, dtype, pad, shift) for n, a in v.items()}
    y = h["r"] if in_place else U.Held(None, dtype, pad, shift, rows, o)
    index, weight, space = Bytes(None, np.int32, pad, shift, rows, k), U.Held(None, F32, pad, shift, rows, k), U.Space()
    p = nn.Experts(h["x"].matrix, h["wr"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, k, act=name,
                   normalize=normalize, residual=h["r"].matrix if residual else None, index=index.matrix, weight=weight.matrix, room=space)
    p.run()
    want, share, ref, bound = V.experts(v["x"], v["wr"], v["wg"], v["wu"], v["wd"], k, name, dtype, normalize, v["r"] if residual else None)
    assert np.array_equal(index.get(), want)
    close("weight", weight.get(), share, V.SHARE * share)
    got = y.get()
    close("y", got, ref, bound)
    if not in_place:
        p.run()
        assert np.array_equal(got, y.get())
    space.check()
    return v, got


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 40])
@pytest.mark.parametrize("d,f,o,e,k", [(1, 1, 1, 1, 1), (8, 16, 8, 3, 2), (33, 17, 40, 5, 5), (64, 128, 64, 8, 2), (200, 130, 72, 16, 4),
                                       (136, 300, 136, 64, 8), (1032, 70, 48, 4, 1)])
@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu"), (BF16, "relu")])
def test_experts(rows, d, f, o, e, k, dtype, name):
    check(rows, d, f, o, e, k, dtype, name, residual=rows % 2 == 0, normalize=k != 4)


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 1), (0, 3)])
@pytest.mark.parametrize("rows", [1, 20])
def test_strides(rows, pad, shift):
    check(rows, 61, 45, 51, 6, 2, BF16, residual=True, pad=pad, shift=shift)
    check(rows, 64, 48, 40, 6, 3, F16, "gelu", residual=True, pad=pad, shift=shift)


@pytest.mark.parametrize("rows,e,k", [(128, 128, 8), (300, 4, 4), (200, 2, 1), (1500, 3, 1), (70, 40, 33), (20, 64, 64), (3, 1024, 64)])
def test_more_pairs_than_a_lot(rows, e, k):
    check(rows, 40, 24, 32, e, k, BF16, residual=True)


def test_y_in_the_place_of_the_residual():
    check(33, 64, 48, 64, 8, 2, BF16, residual=True, in_place=True)


@pytest.mark.parametrize("rows", [1, 5, 33])
def test_equal_experts_go_to_the_lowest_index(rows):
    """Router rows that are copies of each other, zeros of either sign among the logits."""
    def values(v):
        wr = v["wr"].copy()
        wr[[1, 4, 9]] = wr[0]
        wr[[2, 11]] = wr[7]
        wr[5] = 0
        x = v["x"].copy()
        x[0] = 0
        x[rows // 2, ::2] = -0.0
        return dict(wr=wr, x=x)
    for k in (1, 3, 12):
        check(rows, 64, 16, 24, 12, k, BF16, values=values)


def test_logits_that_nearly_agree():
    """Two experts apart by the last bit of one weight, far below what a sum in single precision tells apart."""
    def values(v):
        wr, x = v["wr"].copy(), v["x"].copy()
        wr[3] = abs(wr[3]) + 1
        x[:] = abs(x) + 0.5
        wr[1] = wr[3]
        x[:, 63] = 2.0 ** -30
        wr[1, 63] = wr[3, 63] + 2.0 ** -7
        return dict(wr=wr, x=x)
    check(9, 64, 16, 24, 6, 1, BF16, values=values)


@pytest.mark.parametrize("higher", [1, 3])
def test_logits_apart_by_a_billionth(higher):
    """Two experts' logits of about 64, 2^-37 apart: exact in 64 bits, equal in single precision."""
    def values(v):
        wr, x = v["wr"].copy(), np.ones_like(v["x"])
        wr[[1, 3]] = 1.0
        x[:, 63] = 2.0 ** -30
        wr[higher, 63] = 1 + 2.0 ** -7
        return dict(wr=wr, x=x)
    v, _ = check(9, 64, 16, 24, 6, 1, BF16, values=values)
    assert (V.route(v["x"], v["wr"], 1, True)[0] == higher).all()


def test_tokens_without_numbers_leave_the_others_alone():
    v = make(20, 64, 48, 40, 8, BF16)
    clean = V.experts(v["x"], v["wr"], v["wg"], v["wu"], v["wd"], 2, "silu", BF16)
    for bad in (np.inf, -np.inf, np.nan):
        x = v["x"].copy()
        x[6, 5] = bad
        h = {n: U.Held(a, BF16) for n, a in {**v, "x": x}.items()}
        y, index, weight = U.Held(None, BF16, rows=20, cols=40), Bytes(None, np.int32, rows=20, cols=2), U.Held(None, F32, rows=20, cols=2)
        nn.Experts(h["x"].matrix, h["wr"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, 2, index=index.matrix,
                   weight=weight.matrix, room=U.Space()).run()
        others = [i for i in range(20) if i != 6]
        i, got = index.get(), y.get()
        assert (i >= 0).all() and (i < 8).all() and (i[:, 0] != i[:, 1]).all() and np.array_equal(i[others], clean[0][others])
        close("y", got[others], clean[2][others], clean[3][others])
        assert np.isnan(got[6]).all() and np.isnan(weight.get()[6]).all()


@pytest.mark.parametrize("rows", [1, 5])
def test_subnormal_weights(rows):
    """Which count like any others, and so do the second halves of inner activations, subnormal as a rule."""
    check(rows, 64, 48, 40, 4, 2, F16, name="relu",
          values=lambda v: {"wd": np.random.default_rng(6).integers(-1000, 1001, v["wd"].shape) * 2.0 ** -24, "wg": v["wg"] * 30, "wu": v["wu"] * 30})


@pytest.mark.parametrize("rows", [1, 5])
def test_inner_activations_beyond_the_type(rows):
    """Up to twice float16's largest value they are held as well as others."""
    def values(v):
        # one column of x is 100, and a hidden unit's weights of it give 200 x 250 to 280 x 420: 50000 to 117600
        x, wg, wu = v["x"], 0 * v["wg"], 0 * v["wu"]
        x[:, 0] = 100
        g = np.random.default_rng(7)
        wg[:, 0], wu[:, 0] = 2 + 0.8 * g.random(len(wg)), 2.5 + 1.7 * g.random(len(wu))
        return {"x": x, "wr": np.where(np.arange(64) > 0, v["wr"], 0), "wg": wg, "wu": wu, "wd": v["wd"] * 2.0 ** -10}
    check(rows, 64, 48, 40, 4, 2, F16, name="relu", values=values)


def test_no_rows():
    s = U.Held(np.ones((8, 8)), BF16)
    none = lambda c: nn.Matrix(s.matrix.ptr, 0, c, c, BF16)  # noqa: E731
    nn.Experts(none(8), s.matrix, s.matrix, s.matrix, nn.Matrix(s.matrix.ptr, 8, 1, 1, BF16), none(1), 2).run()


@pytest.mark.parametrize("rows", [1, 30])
def test_a_block_and_its_head(rows):
    """A served block: norm, experts, norm with gate and residual, a 4-bit head on it; each step against 64 bits on what the one before
    gave."""
    d, f, e, k, out, group = 96, 80, 8, 2, 72, 32
    v = make(rows, d, f, d, e, BF16, 5)
    g = np.random.default_rng(8)
    w1, w2 = (U.rounded(1 + 0.2 * g.standard_normal((1, d)), BF16) for _ in range(2))
    w2 = w2[:, :d]
    gate = U.rounded(g.standard_normal((1, d)), BF16)
    head = g.standard_normal((out, d)).astype(np.float32) * d ** -0.5
    code, stored, zero, _ = V.quantised4(head, group, True, BF16)
    h = {n: U.Held(a, BF16) for n, a in v.items()}
    h1, h2, hg = U.Held(w1, BF16), U.Held(w2, BF16), U.Held(gate, BF16)
    n1, y1, y2, n2, y3 = (U.Held(None, BF16, rows=rows, cols=c) for c in (d, d, d, d, out))
    space, n = U.Space(), V.groups(d, group)
    q, s, z = Bytes(None, rows=out, cols=d // 2), U.Held(None, BF16, rows=out, cols=n), Bytes(None, rows=out, cols=n)
    for p in (nn.QuantizeGroups(U.Held(head, F32).matrix, q.matrix, s.matrix, group, zero=z.matrix),
              nn.BlockNorm(residual=h["x"].matrix, n=n1.matrix, w_pre=h1.matrix),
              nn.Experts(n1.matrix, h["wr"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y1.matrix, k, room=space),
              nn.BlockNorm(x=y1.matrix, residual=h["x"].matrix, gate=hg.matrix, gate_act="sigmoid", scale=0.7, y=y2.matrix, n=n2.matrix, w_pre=h2.matrix),
              nn.Q4Linear(n2.matrix, q.matrix, s.matrix, y3.matrix, group, zero=z.matrix, room=space)):
        (p.forward if isinstance(p, nn.BlockNorm) else p.run)()
    a = n1.get()
    close("n", a, *V.block_norm(BF16, BF16, r=v["x"], w_pre=w1[0])["n"])
    b = y1.get()
    _, _, ref, bound = V.experts(a, v["wr"], v["wg"], v["wu"], v["wd"], k, "silu", BF16)
    close("experts", b, ref, bound)
    want = V.block_norm(BF16, BF16, x=b, r=v["x"], gate=gate, per=rows, act="sigmoid", scale=0.7, w_pre=w2[0])
    close("y", y2.get(), *want["y"])
    c = n2.get()
    close("n", c, *want["n"])
    close("head", y3.get(), *V.q4_linear(c, code, U.value(stored, BF16), zero, group, BF16, True))
    space.check()
