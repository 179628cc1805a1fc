"""Calls of the norms, 4-bit products and experts that reach no GPU: batches of no rows, whose matrices have no address."""
import numpy as np
import pytest

from b2ctrain_amd import nn
from tests.test_dense_host import ADDRESS, M

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def none(cols, dtype=BF16):
    return nn.Matrix(0, 0, cols, cols, dtype)


@pytest.mark.parametrize("form", ["both", "x", "residual", "gate"])
def test_norms_of_no_rows(form):
    w = nn.Matrix(ADDRESS, 1, 40, 40, BF16)
    given = dict(x=none(40) if form != "residual" else None, residual=none(40) if form != "x" else None)
    if form != "residual":
        given.update(y=none(40), post=True, w_post=w)
    if form == "gate":
        given.update(gate=none(40), rows_per_gate=3, gate_act="sigmoid")
    p = nn.BlockNorm(n=none(40), w_pre=w, **given)
    p.forward()
    for dn in (none(40), None):
        p.gradients(dy=none(40), dn=dn, dx=none(40) if form != "residual" else None, dresidual=none(40), dgate=none(40) if form == "gate" else None)
        p.backward()


def test_gradients_of_no_rows_are_refused_as_of_some():
    """What no number of rows makes right."""
    p = nn.BlockNorm(x=none(40), residual=none(40), n=none(40))
    p.gradients(dn=none(40), dx=none(40))
    p.grad.dw_post = ADDRESS  # without `post`
    with pytest.raises(ValueError, match="invalid arguments"):
        p.backward()
    p.grad.dw_post, p.grad.grad_dtype = None, 7
    with pytest.raises(ValueError, match="invalid arguments"):
        p.backward()
    p.args.kind = 5
    with pytest.raises(ValueError, match="invalid arguments"):
        p.forward()


def test_products_and_experts_of_no_rows():
    nn.QuantizeGroups(none(40), none(20, nn.U8), none(2), 32, values=none(40)).run()
    nn.Q4Linear(none(40), M(8, 20, nn.U8), M(8, 2), none(8), 32).run()
    nn.Experts(none(40), M(4, 40), M(32, 40), M(32, 40), M(4 * 40, 8), none(40), 2, residual=none(40), index=none(2, nn.I32), weight=none(2, F32)).run()
