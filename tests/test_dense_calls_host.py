"""Calls of the dense operators that differ from the usual ones in one thing: an alignment, a buffer's place, a size at the end of
its range. What can be seen of them without a GPU."""
import ctypes as C

import pytest
import torch

from b2ctrain_amd import _native, nn
from tests import dense_bounds as B
from tests import dense_util as U
from tests.test_dense_host import ADDRESS, M, Room


def column(n, ptr=ADDRESS):
    return nn.Matrix(ptr, n, 1, 1, nn.F32)


@pytest.mark.parametrize("rows,di,f,ld,pitch", [(64, 144, 256, 144, 256), (64, 256, 320, 272, 256), (200, 48, 1040, 48, 128)])
def test_i8_block_copies_both_input_weights_or_none(rows, di, f, ld, pitch):
    """The tiles read both with one distance between rows, so a weight beside one that is copied is copied too."""
    def room(gate, up):
        p = nn.I8FeedForward(M(rows, di), M(f, di, nn.I8, ld, ADDRESS + gate), column(f), M(f, di, nn.I8, ld, ADDRESS + up), column(f),
                             M(di, f, nn.I8), column(di), M(rows, di), room=Room())
        return p.args.workspace_bytes

    assert room(0, 8) == room(8, 0) == room(8, 8) == room(0, 0) + 2 * f * pitch


def linear(scale, room=Room()):
    return nn.I8Linear(M(4, 5), M(6, 5, nn.I8), scale, M(4, 6), room=room)


@pytest.mark.parametrize("scale", [
    torch.ones(6), nn.Matrix(ADDRESS, 6, 1, 9, nn.F32), nn.Matrix(ADDRESS, 2, 3, 4, nn.F32), nn.Matrix(0, 6, 1, 1, nn.F32),
    nn.Matrix(ADDRESS, 6, 1, 1, nn.BF16), 3, None, [1.0] * 6], ids=str)
def test_scales_have_to_lie_on_the_gpu_next_to_each_other(scale):
    with pytest.raises(ValueError, match="scale"):
        linear(scale)
    with pytest.raises(ValueError, match="scale"):
        nn.QuantizeRows(M(6, 5), M(6, 5, nn.I8), scale)
    for at in range(3):
        s = [scale if i == at else column(6) for i in range(3)]
        with pytest.raises(ValueError, match="s_"):
            nn.I8FeedForward(M(4, 5), M(6, 5, nn.I8), s[0], M(6, 5, nn.I8), s[1], M(6, 6, nn.I8), s[2], M(4, 6), room=Room())


def test_scales_that_are_taken():
    for scale in (column(6), nn.Matrix(ADDRESS, 1, 6, 6, nn.F32), nn.Matrix(ADDRESS, 1, 6, 20, nn.F32), nn.Matrix(ADDRESS, 2, 3, 3, nn.F32)):
        assert linear(scale).args.w_scale == ADDRESS


def test_workspace_has_to_lie_on_the_gpu_and_be_large_enough():
    need = linear(column(6)).args.workspace_bytes

    class Bytes(Room):
        is_cuda = True

        def __init__(self, nbytes):
            self.nbytes = nbytes

    linear(column(6), lambda n: Bytes(n))
    for room in (lambda n: torch.empty(n, dtype=torch.uint8), lambda n: Bytes(need - 1), lambda n: None, lambda n: bytearray(n)):
        with pytest.raises(ValueError, match="workspace"):
            linear(column(6), room)


@pytest.mark.parametrize("entry,args", [("b2c_feed_forward", nn.FfnArgs), ("b2c_feed_forward_backward", nn.FfnGradArgs),
                                        ("b2c_i8_linear", nn.I8LinearArgs), ("b2c_i8_feed_forward", nn.I8FfnArgs)])
def test_a_null_handle_or_argument_is_an_error(entry, args):
    L = _native.lib()
    fn, p = getattr(L, entry), C.c_void_p
    fn.argtypes = [p, p, C.c_int, p] if entry == "b2c_feed_forward" else [p, p, p]
    more = (1, None) if entry == "b2c_feed_forward" else (None,)
    L.b2c_dense_create.restype, L.b2c_dense_destroy.argtypes = p, [p]
    d, some = L.b2c_dense_create(), args()
    try:
        for handle, a in ((None, C.addressof(some)), (d, None), (None, None)):
            assert fn(handle, a, *more) != 0 and b"null" in L.b2c_last_error()
    finally:
        L.b2c_dense_destroy(d)
        L.b2c_dense_destroy(None)


@pytest.mark.parametrize("rows,di,f,do", [(1500, 2792, 7008, 2792), (3193, 1496, 5392, 48), (4545, 3336, 2320, 369), (5204, 3664, 128, 2832),
                                          (86, 3949, 4311, 20), (40, 64, 96, 64), (3, 64, 96, 64)])
def test_block_workspace_is_the_same_with_and_without_kept_values(rows, di, f, do):
    """A call that answers may follow one that trains in the same workspace, and the other way round."""
    def room(train):
        return nn.FeedForward(M(rows, di), M(f, di), M(f, di), M(do, f), M(rows, do), train=train, room=Room()).args.workspace_bytes

    assert room(False) == room(True)


@pytest.mark.parametrize("rows,di,f,do,kept", [
    (40, 96, 8192, 96, True), (33, 128, 1 << 20, 128, True), (2000, 128, 2048, 128, True), (8000, 64, 256, 64, True), (40, 96, 64, 96, False),
    (16384, 96, 8192, 96, False), (1_000_000, 64, 256, 64, False), (1_000_000, 64, 256, 129, True), (1_000_000, 129, 256, 3, True),
    (32, 64, 64, 64, True)])
def test_a_block_is_a_head_where_its_rows_fill_the_device(rows, di, f, do, kept):
    """A head keeps nothing for its backward pass. Its workgroups share out rows alone and each passes over the whole hidden width."""
    a = nn.FfnArgs(rows=rows, d_in=di, d_hidden=f, d_out=do, dtype=nn.BF16)
    assert (nn._lib().b2c_ffn_saved_bytes(C.byref(a)) > 0) == kept


@pytest.mark.parametrize("dtype,name", [(nn.BF16, "silu"), (nn.F16, "gelu")])
def test_the_gradients_bound_sees_one_rounding_more(dtype, name):
    """The roundings that the block makes stay within the bound; with g and u rounded too some outputs of each kind do not, with the
    factors of dg and du some that come from those."""
    past = {(k, what): 0 for k in ("dx", "dw_gate", "dw_up", "dw_down") for what in ("factors", "inputs") if (k, what) != ("dw_down", "factors")}
    for seed, sizes in enumerate(B.SINGLE * 4):
        x, wg, wu, wd, dy = B.make(*sizes, dtype, seed)
        m = U.mask(sizes[0], sizes[3], 0.2, 7, 5)
        ref, bound = B.grads_bound(x, wg, wu, wd, name, dtype, dy, m)
        got = B.rounded_grads(x, wg, wu, wd, name, dtype, dy, m)
        for k in ref:
            assert (abs(got[k] - ref[k]) <= bound[k]).all(), (sizes, k)
        for k, what in past:
            more = B.rounded_grads(x, wg, wu, wd, name, dtype, dy, m, **{what: True})
            past[k, what] += (abs(more[k] - ref[k]) > bound[k]).sum()
    assert all(past.values()), past


def test_accumulating_with_no_weight_gradient_wanted_is_taken():
    """A loop that accumulates may pass through a block whose weights are frozen."""
    f = nn.FeedForward(M(8, 16), M(32, 16), M(32, 16), M(24, 32), M(8, 24), train=True, room=Room())
    f.gradients(M(8, 24), dx=M(8, 16), accumulate=True, room=Room())
    assert f.grad.accumulate == 1 and f.grad.grad_dtype == nn.F32  # which is what the launcher takes with it
