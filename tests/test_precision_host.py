"""That the measure of precision tells kernels apart which round where they need not: the oracle with such a rounding planted in it."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests import dense_util as U
from tests import more_util as V
from tests import precision as P

F16, BF16 = nn.F16, nn.BF16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,n,group", [(5, 2050, 1040, 32), (33, 515, 900, 64), (17, 128, 2048, 128)])
def test_a_rounding_too_many_in_products_is_seen(rows, k, n, group, dtype):
    x, code, scale, zero, w = P.weights4(rows, k, n, group, True, dtype)
    want = x @ w.T
    wide = lambda v: np.repeat(v, group, axis=1)[:, :k].astype(np.float64)  # noqa: E731
    assert P.excess(U.rounded(want, dtype), want, dtype) == 1
    assert P.excess(U.rounded(want + want * np.random.default_rng(0).uniform(-1, 1, want.shape) * 2.0 ** -20, dtype), want, dtype) < P.MOST
    assert P.excess(U.rounded(x @ U.rounded(w, dtype).T, dtype), want, dtype) > 1.2  # the weights, once
    part = lambda i, v: v[:, i * group:(i + 1) * group]  # noqa: E731
    sums = sum(U.rounded(part(i, x) @ part(i, code - wide(zero)).T, dtype) * scale[:, i] for i in range(V.groups(k, group)))
    assert P.excess(U.rounded(sums, dtype), want, dtype) > 1.2  # each group's sum


@pytest.mark.parametrize("dtype,name", [(BF16, "silu"), (F16, "gelu"), (F16, "silu"), (BF16, "relu")])
@pytest.mark.parametrize("rows,d,f,o,e,k", [(7, 64, 128, 512, 8, 2), (40, 136, 300, 1000, 64, 8), (16, 200, 7, 800, 4, 2)])
def test_inner_activations_rounded_once_are_seen(rows, d, f, o, e, k, dtype, name):
    from tests.test_gpu_experts import make
    v = make(rows, d, f, o, e, dtype)
    want = P.experts(v, k, name)
    assert np.array_equal(want, V.experts(v["x"], v["wr"], v["wg"], v["wu"], v["wd"], k, name, dtype)[2])
    by = lambda held: U.rounded(P.experts(v, k, name, held), dtype)  # noqa: E731
    first = lambda h: U.rounded(h, dtype)  # noqa: E731
    assert P.excess(by(lambda h: first(h) + first(h - first(h))), want, dtype) < P.MOST
    assert P.excess(by(first), want, dtype) > 1.2
