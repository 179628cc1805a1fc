"""The norms, gate and residual sum between two blocks, and their gradients, against their restatement in 64 bits (more_util.py)."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests.gpu_harness import emit
from tests.test_gpu_dense import close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def make(rows, d, dtype, w_dtype, gate_rows, seed):
    g = np.random.default_rng(seed)
    q = lambda k=1.0, n=rows, add=0.0, t=dtype: U.rounded(g.standard_normal((n, d)) * k + add, t)  # noqa: E731
    return dict(x=q(0.5), r=q(2.0), gate=q(n=gate_rows) if gate_rows else None, w_post=q(0.2, 1, 1.0, w_dtype)[0],
                w_pre=q(0.2, 1, 1.0, w_dtype)[0], dy=q(0.1), dn=q(0.1))


def check(rows, d, dtype, w_dtype=None, kind="rms", per=0, act="none", post=True, weights=True, residual=True, x=True, n=True, y=True,
          use_dy=True, use_dn=True, pad=0, shift=0, grad=None, accumulate=False, seed=0, scale=0.5, values=None):
    w_dtype = dtype if w_dtype is None else w_dtype
    grad = w_dtype if grad is None else grad
    emit(f"block norm {rows} x {d} type {dtype} weights {w_dtype} {kind} per {per} {act} post {post} pad {pad} shift {shift}")
    v = make(rows, d, dtype, w_dtype, -(-rows // per) if per else 0, seed + rows + d)
    if values:
        v.update(values(v))
    hold = lambda a, t=dtype: U.Held(a, t, pad, shift)  # noqa: E731
    h = {k: hold(a) for k, a in v.items() if a is not None and k not in ("w_post", "w_pre")}
    w = {k: U.Held(v[k][None], w_dtype, 0, shift) for k in ("w_post", "w_pre")} if weights else {}
    if not post:
        w.pop("w_post", None)
    if not n:
        w.pop("w_pre", None)
    out = {k: U.Held(None, dtype, pad, shift, rows, d) for k in ("y", "n", "dx", "dresidual")}
    given = dict(x=h["x"].matrix if x else None, residual=h["r"].matrix if residual else None, gate=h["gate"].matrix if per else None,
                 rows_per_gate=per or None, gate_act=act, post=post, kind=kind, scale=scale, eps=1e-5,
                 **{k: m.matrix for k, m in w.items()})
    p = nn.BlockNorm(y=out["y"].matrix if y and x else None, n=out["n"].matrix if n else None, **given)
    want = V.block_norm(dtype, w_dtype, x=v["x"] if x else None, r=v["r"] if residual else None, gate=v["gate"], per=per or 1, act=act,
                        post=post, w_post=v["w_post"] if "w_post" in w else None, w_pre=v["w_pre"] if "w_pre" in w else None, kind=kind,
                        eps=1e-5, scale=scale, want_n=n, dy=v["dy"] if use_dy else None, dn=v["dn"] if use_dn and n else None,
                        grad_dtype=grad)
    p.forward()
    for k in ("y", "n"):
        if k == "y" and (not y or not x) or k == "n" and not n:
            continue
        close(k, out[k].get(), *want[k])
    space = U.Space()
    grads = {"dresidual": out["dresidual"]}
    if x:
        grads["dx"] = out["dx"]
    if per:
        grads["dgate"] = U.Held(None, dtype, pad, shift, v["gate"].shape[0], d)
    start = {}
    for k in ("dw_post", "dw_pre"):
        if k in want:
            start[k] = U.rounded(np.random.default_rng(3).standard_normal((1, d)), grad)
            grads[k] = U.Held(start[k], grad, 0, shift)
    p.gradients(dy=h["dy"].matrix if use_dy else None, dn=h["dn"].matrix if use_dn and n else None, accumulate=accumulate, room=space,
                **{k: m.matrix for k, m in grads.items()})
    got = []
    for _ in range(2):
        p.backward()
        got.append({k: m.get() for k, m in grads.items()})
        if accumulate:
            break
    for k, m in got[0].items():
        ref, bound = want[k]
        if k in start:
            m = m[0]
            if accumulate:
                ref, bound = ref + start[k][0], bound + U.F32_SUM * abs(ref + start[k][0])
        close(k, m, ref, bound)
        assert len(got) == 1 or np.array_equal(got[0][k], got[1][k]), f"{k}: another result from the same call"
    space.check()
    return p, h, out, grads


# Widths on both sides of every team's size, for 16 bits (8 values a lane) and 32 (4).
@pytest.mark.parametrize("d", [1, 3, 8, 45, 64, 65, 128, 200, 256, 512, 513, 1000, 2048, 2049, 4096, 4100, 8192, 8200, 16384])
@pytest.mark.parametrize("dtype,kind", [(BF16, "rms"), (F16, "layer"), (F32, "layer"), (F32, "rms")])
def test_widths(d, dtype, kind):
    check(19, d, dtype, kind=kind)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 300, 5000])
@pytest.mark.parametrize("d", [24, 64, 600])
@pytest.mark.parametrize("per", [0, 1, 7, 10000])
@pytest.mark.parametrize("dtype,w_dtype,act", [(BF16, F32, "sigmoid"), (F16, F16, "none"), (F32, F32, "sigmoid")])
def test_gates(rows, d, per, dtype, w_dtype, act):
    check(rows, d, dtype, w_dtype, per=per, act=act if per else "none")


@pytest.mark.parametrize("rows,d,per", [(4000, 32, 1), (4000, 32, 2), (4000, 32, 3), (4000, 32, 1999), (4000, 32, 4000), (600, 3000, 2),
                                        (600, 3000, 299), (600, 3000, 600), (9000, 8, 1), (9000, 8, 4), (40, 9000, 13)])
@pytest.mark.parametrize("dtype,kind", [(BF16, "layer"), (F32, "rms")])
def test_shared_gates(rows, d, per, dtype, kind):
    check(rows, d, dtype, F32, kind=kind, per=per, act="sigmoid")


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 1), (0, 3), (24, 8)])
@pytest.mark.parametrize("d", [45, 64, 1000, 2048])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(pad, shift, d, dtype):
    check(37, d, dtype, per=5, act="sigmoid", kind="layer", pad=pad, shift=shift)


FORMS = [dict(post=False), dict(weights=False), dict(residual=False), dict(n=False, use_dn=False), dict(x=False, post=False),
         dict(y=False), dict(use_dy=False), dict(use_dn=False), dict(post=False, n=False, use_dn=False), dict(post=False, weights=False, residual=False),
         dict(x=False, post=False, weights=False, use_dy=False)]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(f"{k}={v}" for k, v in f.items()))
@pytest.mark.parametrize("d", [40, 2500])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_forms(form, d, kind):
    check(50, d, BF16, kind=kind, per=0 if form.get("x") is False else 3, **form)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,d", [(3, 40), (700, 64), (300, 2600)])
def test_weight_gradients_in_single_precision(rows, d, accumulate):
    check(rows, d, BF16, BF16, grad=F32, accumulate=accumulate)


def test_many_rows():
    check(70001, 64, BF16, F32, per=70001)
    check(70001, 33, F16, F16, per=1, act="sigmoid", kind="layer")


def test_rows_far_from_zero():
    """A layer norm of rows whose mean is a thousand times their spread."""
    for d in (64, 600, 5000):
        check(20, d, F32, kind="layer", values=lambda v: dict(x=U.rounded(v["x"] + 500, F32), r=U.rounded(v["r"] - 2000, F32)))


def test_large_offsets_of_dresidual_in_dy():
    """dresidual over dy and dx over dn, y over residual and n over x."""
    rows, d = 100, 200
    v = make(rows, d, BF16, BF16, 0, 5)
    want = V.block_norm(BF16, BF16, x=v["x"], r=v["r"], post=True, w_post=v["w_post"], w_pre=v["w_pre"], scale=0.5, dy=v["dy"], dn=v["dn"])
    h = {k: U.Held(v[k], BF16) for k in ("x", "r", "dy", "dn")}
    w = {k: U.Held(v[k][None], BF16) for k in ("w_post", "w_pre")}
    p = nn.BlockNorm(x=h["x"].matrix, residual=h["r"].matrix, n=h["x"].matrix, y=h["r"].matrix, post=True, scale=0.5,
                     **{k: m.matrix for k, m in w.items()})
    p.gradients(dy=h["dy"].matrix, dn=h["dn"].matrix, dx=h["dn"].matrix, dresidual=h["dy"].matrix, room=U.Space())
    p.backward()
    p.forward()
    for k, m in (("dresidual", "dy"), ("dx", "dn"), ("y", "r"), ("n", "x")):
        close(k, h[m].get(), *want[k])


def test_rows_that_hold_no_number():
    """A row with a NaN is NaN throughout; one with an infinity is infinitely large, so that its other values become zeros and the infinity
    itself NaN. The rows around them get nothing of it; a row of zeros is zeros."""
    rows, d = 70, 96
    v = make(rows, d, F32, F32, 0, 9)
    clean = V.block_norm(F32, F32, x=v["x"], r=v["r"], post=True, scale=1.0, dy=v["dy"], dn=v["dn"])
    for bad in (np.inf, -np.inf, np.nan):
        x, r = v["x"].copy(), v["r"].copy()
        x[13, 5], r[50, 95] = bad, bad
        x[20], r[20] = 0, 0
        h = {k: U.Held(a, F32) for k, a in (("x", x), ("r", r), ("dy", v["dy"]), ("dn", v["dn"]))}
        out = {k: U.Held(None, F32, rows=rows, cols=d) for k in ("y", "n", "dx", "dresidual")}
        p = nn.BlockNorm(x=h["x"].matrix, residual=h["r"].matrix, y=out["y"].matrix, n=out["n"].matrix, post=True)
        p.gradients(dy=h["dy"].matrix, dn=h["dn"].matrix, dx=out["dx"].matrix, dresidual=out["dresidual"].matrix, room=U.Space())
        p.forward()
        p.backward()
        others = [i for i in range(rows) if i not in (13, 20, 50)]
        for k, m in out.items():
            got = m.get()
            close(k, got[others], clean[k][0][others], clean[k][1][others])
            if k in ("y", "n"):
                assert not got[20].any()
                assert np.isnan(got[13, 5] if k == "y" or np.isinf(bad) else got[13]).all()
                assert not np.isfinite(got[50, 95]) and (k == "y" or np.isnan(got[50, 95]))
                assert k == "y" and np.array_equal(got[13, 6:], r[13, 6:]) or k == "n" or not np.isinf(bad)


def test_gradients_along_their_direction():
    """L = sum(y dy + n dn): its difference along the sign of each gradient is the gradient's sum of magnitudes. In single precision, with a
    step of 2^-10: the third derivatives leave less than a thousandth of it, the sums' roundings less than that."""
    rows, d, per, e = 60, 80, 7, 2.0 ** -10
    v = make(rows, d, F32, F32, -(-rows // per), 2)

    def loss(v):
        h = {k: U.Held(v[k], F32) for k in ("x", "r", "gate")}
        w = {k: U.Held(v[k][None], F32) for k in ("w_post", "w_pre")}
        y, n = (U.Held(None, F32, rows=rows, cols=d) for _ in range(2))
        nn.BlockNorm(x=h["x"].matrix, residual=h["r"].matrix, gate=h["gate"].matrix, rows_per_gate=per, gate_act="sigmoid", post=True,
                     y=y.matrix, n=n.matrix, scale=0.5, **{k: m.matrix for k, m in w.items()}).forward()
        return (y.get() * v["dy"]).sum() + (n.get() * v["dn"]).sum()

    h = {k: U.Held(v[k], F32) for k in ("x", "r", "gate", "dy", "dn")}
    w = {k: U.Held(v[k][None], F32) for k in ("w_post", "w_pre")}
    g = {k: U.Held(None, F32, rows=v[k].shape[0], cols=d) for k in ("x", "r", "gate")}
    gw = {k: U.Held(None, F32, rows=1, cols=d) for k in w}
    p = nn.BlockNorm(x=h["x"].matrix, residual=h["r"].matrix, gate=h["gate"].matrix, rows_per_gate=per, gate_act="sigmoid", post=True,
                     n=U.Held(None, F32, rows=rows, cols=d).matrix, scale=0.5, **{k: m.matrix for k, m in w.items()})
    p.gradients(dy=h["dy"].matrix, dn=h["dn"].matrix, dx=g["x"].matrix, dresidual=g["r"].matrix, dgate=g["gate"].matrix,
                dw_post=gw["w_post"].matrix, dw_pre=gw["w_pre"].matrix, room=U.Space())
    p.backward()
    for k in ("x", "r", "gate", "w_post", "w_pre"):
        grad = g[k].get() if k in g else gw[k].get()[0]
        side = []
        for t in (e, -e):
            moved = dict(v)
            moved[k] = v[k] + t * np.sign(grad)
            side.append(loss(moved))
        assert abs((side[0] - side[1]) / (2 * e) - abs(grad).sum()) < 2e-3 * abs(grad).sum(), k


def test_no_rows():
    v = make(1, 40, F32, F32, 0, 1)
    h = U.Held(v["x"], F32)
    none = lambda: nn.Matrix(h.matrix.ptr, 0, 40, 40, F32)  # noqa: E731
    w = U.Held(v["w_pre"][None], F32)
    p = nn.BlockNorm(x=none(), residual=none(), y=none(), n=none(), post=True)
    p.forward()
    for accumulate in (True, False):
        p.gradients(dy=none(), dn=none(), dx=none(), dw_pre=w.matrix, accumulate=accumulate, room=U.Space())
        p.backward()
        assert np.array_equal(w.get()[0], v["w_pre"] if accumulate else np.zeros(40))
