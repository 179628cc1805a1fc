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
