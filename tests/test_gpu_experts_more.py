"""How exactly the experts' outputs and inner activations are held."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import precision as P
from tests.gpu_harness import emit
from tests.test_gpu_experts import make
from tests.test_gpu_q4 import Bytes

pytestmark = pytest.mark.gpu

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def run(v, k, dtype, name, residual=False):
    rows, o = v["r"].shape
    h = {n: U.Held(a, dtype) for n, a in v.items()}
    y, space = U.Held(None, dtype, rows=rows, cols=o), U.Space()
    nn.Experts(h["x"].matrix, h["wr"].matrix, h["wg"].matrix, h["wu"].matrix, h["wd"].matrix, y.matrix, k, act=name,
               residual=h["r"].matrix if residual else None, room=space).run()
    space.check()
    return y.get()


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 40, 150])
@pytest.mark.parametrize("d,f,o,e,k", [(64, 128, 512, 8, 2), (136, 300, 400, 64, 8), (1000, 1365, 350, 10, 3), (200, 7, 800, 4, 2),
                                       (5, 900, 640, 5, 5), (72, 130, 350, 300, 4)])
@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu"), (F16, "silu"), (BF16, "relu")])
def test_outputs_are_as_exact_as_their_rounding(rows, d, f, o, e, k, dtype, name):
    """So the inner activations enter as more than one value of 16 bits, whose second one is subnormal in half precision as a rule."""
    emit(f"experts {rows} x {d}-{f}-{o}, {k} of {e}, type {dtype} {name}")
    v = make(rows, d, f, o, e, dtype)
    want = P.experts(v, k, name)
    for residual in (False, True):
        assert P.excess(run(v, k, dtype, name, residual), want + v["r"] * residual, dtype) < (P.MOST if rows * o > 2000 else 1.2)


def pairs_of_units(rows, n, dtype, w_gate, w_up, c):
    """Outputs that are the difference of two hidden units: relu(w_gate x) (w_up x) with x = (1, 2^-8, 0 ..), and c."""
    f, d = 2 * n, 16
    v = dict(x=np.zeros((rows, d)), wr=np.zeros((1, d)), wg=np.zeros((f, d)), wu=np.zeros((f, d)), wd=np.zeros((n, f)), r=np.zeros((rows, n)))
    v["x"][:, 0], v["x"][:, 1] = 1, 2.0 ** -8
    v["wg"][0::2, 0], v["wg"][0::2, 1], v["wu"][0::2, 0] = w_gate[0], w_gate[1], w_up
    v["wg"][1::2, 0], v["wu"][1::2, 0] = 1, c
    v["wd"][np.arange(n), 2 * np.arange(n)], v["wd"][np.arange(n), 2 * np.arange(n) + 1] = 1, -1
    return v


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("dtype,unit", [(BF16, 2.0 ** -17), (F16, 2.0 ** -23)])
def test_inner_activations_are_held_as_two_values(rows, dtype, unit):
    """An inner activation less its own rounding to 16 bits leaves what the second value holds. The product of two 16-bit numbers has no more
    bits than the two values, and comes out to the bit; one of more bits is off by at most `unit` of itself."""
    g, n = np.random.default_rng(rows), 400
    a, b = U.rounded(g.uniform(4, 8, n), dtype), U.rounded(g.uniform(16, 32, n), dtype)
    h = a * b
    c = U.rounded(h, dtype)
    assert (h != c).mean() > 0.5
    got = run(pairs_of_units(rows, n, dtype, (a, 0 * a), b, c), 1, dtype, "relu")
    assert np.array_equal(got, np.tile(h - c, (rows, 1)))
    a2 = U.rounded(g.uniform(1, 2, n), dtype)
    h = (a + a2 * 2.0 ** -8) * b
    c = U.rounded(h, dtype)
    got = run(pairs_of_units(rows, n, dtype, (a, a2), b, c), 1, dtype, "relu")
    # besides: two roundings in single precision, and y's own
    off = abs(got - (h - c)) - U.UNIT[dtype] * abs(h - c) - 2 * 2.0 ** -24 * h
    assert (off <= unit * h).all()


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_inner_activations_between_once_and_twice_the_largest_value(rows):
    """The first value stays at half precision's largest, 65504, and the second takes the rest, rounded to its own 11 bits: off by at most 16."""
    g, n = np.random.default_rng(rows), 300
    a, b = U.rounded(g.uniform(256, 300, n), F16), U.rounded(g.uniform(257, 420, n), F16)
    h, c = a * b, np.full(n, 65504.0)
    assert h.min() > 65504 and h.max() < 2 * 65504 and h.max() > 120000
    got = run(pairs_of_units(rows, n, F16, (a, 0 * a), b, c), 1, F16, "relu")
    assert np.array_equal(got, np.tile(U.rounded(h - c, F16), (rows, 1))) and (abs(got - (h - c)) <= 16).all()
    # and beyond twice the largest they are infinite (of one output, since a weight of zero makes NaN of an infinite unit)
    got = run(pairs_of_units(rows, 1, F16, (a[:1], 0 * a[:1]), b[:1] + 256, c[:1]), 1, F16, "relu")
    assert (got == np.inf).all()
