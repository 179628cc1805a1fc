"""The dense operators' plans and refusals, which need no GPU, and the tests' own restatement of them: dropout's bits
against the published test vectors, the block's gradients against differences."""
import ctypes as C

import numpy as np
import pytest

from b2ctrain_amd import _native, nn
from tests import dense_util as U


def test_philox_published_vectors():
    """Known answers of Philox4x32-10 (published with the paper's reference implementation)."""
    full = 0xFFFFFFFF
    for c, k, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((full,) * 4, (full,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(U.philox(np.array([c], np.uint64), k)[0]) == want


@pytest.mark.parametrize("name", ["silu", "gelu", "relu"])
def test_block_gradients_against_differences(name):
    """The oracle's gradients against central differences in 64 bits: off by the step squared and by rounding / step."""
    g = np.random.default_rng(5)
    x, wg, wu, wd = (g.standard_normal(s) for s in ((5, 7), (11, 7), (11, 7), (6, 11)))
    dy, m = g.standard_normal((5, 6)), U.mask(5, 6, 0.3, 9, 4)
    grads = U.block_grads(x, wg, wu, wd, name, dy, m)
    h = 1e-5
    for key, arr in (("dx", x), ("dw_gate", wg), ("dw_up", wu), ("dw_down", wd)):
        for idx in zip(*(g.integers(0, n, 12) for n in arr.shape)):
            keep = arr[idx]
            vals = []
            for s in (h, -h):
                arr[idx] = keep + s
                vals.append((U.block(x, wg, wu, wd, name, None, m) * dy).sum())
            arr[idx] = keep
            assert abs((vals[0] - vals[1]) / (2 * h) - grads[key][idx]) < 1e-6 * (1 + abs(grads[key][idx])), (key, idx)


def test_mask_counts_and_scale():
    m = U.mask(200, 333, 0.25, 123, 7)
    assert abs((m > 0).mean() - 0.75) < 4 * np.sqrt(0.75 * 0.25 / m.size)
    assert set(np.unique(m)) == {0.0, 65536 / (65536 - 16384)}


ADDRESS = 1 << 20  # never read: every call here is refused before a launch


def M(rows, cols, dtype=nn.BF16, ld=None, ptr=ADDRESS):
    return nn.Matrix(ptr, rows, cols, ld or cols, dtype)


class Room:
    def __call__(self, n):
        return self

    def data_ptr(self):
        return ADDRESS


def ffn(**kw):
    a = dict(x=M(8, 16), w_gate=M(32, 16), w_up=M(32, 16), w_down=M(24, 32), y=M(8, 24), train=True, room=Room())
    a.update(kw)
    return nn.FeedForward(**a)


@pytest.mark.parametrize("kw", [
    dict(x=M(8, 16, nn.F32)), dict(w_gate=M(32, 15)), dict(w_up=M(31, 16)), dict(w_down=M(24, 33)), dict(y=M(8, 25)),
    dict(y=M(7, 24)), dict(w_down=M(24, 32, nn.F16)), dict(residual=M(8, 23)), dict(act="tanh"), dict(p=1.0), dict(p=-0.1),
    dict(p=float("nan")), dict(p=0.999999), dict(room=None), dict(w_up=M(32, 16, ld=20)), dict(x=M(8, 16, ld=8)),
    dict(x=M(8, 16, ptr=0)), dict(x=np.zeros((8, 16), np.float16)), dict(x=3)])
def test_feed_forward_plan_refuses(kw):
    with pytest.raises(ValueError):
        ffn(**kw)


@pytest.mark.parametrize("kw", [
    dict(dy=M(8, 23)), dict(dx=M(8, 15)), dict(dw_gate=M(32, 17)), dict(dw_down=M(24, 31)), dict(dw_gate=M(32, 16, nn.F16)),
    dict(dw_gate=M(32, 16), dw_up=M(32, 16, nn.F32)), dict(dw_gate=M(32, 16), accumulate=True),
    dict(dw_gate=M(32, 16), dw_up=M(32, 16, ld=18))])
def test_gradient_plan_refuses(kw):
    f = ffn()
    with pytest.raises(ValueError):
        f.gradients(**{"dy": M(8, 24), "room": Room(), **kw})
    with pytest.raises(ValueError):
        ffn(train=False).gradients(M(8, 24), room=Room())
    with pytest.raises(ValueError):
        f.backward(0)


def refused(fn, args, **kw):
    """The launcher itself, past the plan's checks."""
    for k, v in kw.items():
        obj = args
        *path, last = k.split("__")
        for p in path:
            obj = getattr(obj, p)
        setattr(obj, last, v)
    return fn(C.byref(args), None) == 1


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(d_in=0), dict(d_hidden=0), dict(d_out=0), dict(dtype=0), dict(dtype=3),
    dict(act=3), dict(act=-1), dict(p=1.0), dict(p=-1e-3), dict(x=None), dict(x=ADDRESS + 1), dict(w_gate=None),
    dict(w_up=None), dict(w_down=None), dict(y=None), dict(ldx=15), dict(ld_in=15), dict(ld_out=31), dict(ldy=23),
    dict(workspace=None), dict(workspace=ADDRESS + 8), dict(workspace_bytes=16), dict(saved=ADDRESS + 2),
    dict(residual=ADDRESS, ldr=23)])
def test_forward_launcher_refuses(kw):
    f = ffn()
    assert refused(nn._lib().b2c_hip_ffn_forward, f.args, **kw)


@pytest.mark.parametrize("width", ["d_in", "d_hidden", "d_out"])
def test_launchers_refuse_widths_beyond_their_offsets(width):
    """256 rows of 2^22 16-bit values are the 2 GiB that a copy's offset spans, and a gradient's rows hold two widths."""
    wide = {width: (1 << 20) + 1, "ldx": 1 << 21, "ld_in": 1 << 21, "ld_out": 1 << 21, "ldy": 1 << 21, "workspace_bytes": 1 << 62}
    assert refused(nn._lib().b2c_hip_ffn_forward, ffn().args, **wide)
    f = ffn()
    f.gradients(M(8, 24), dx=M(8, 16), dw_gate=M(32, 16), dw_up=M(32, 16), dw_down=M(24, 32), room=Room())
    ld = {k: 1 << 21 for k in ("lddy", "lddx", "ld_din", "ld_dout")}
    assert refused(nn._lib().b2c_hip_ffn_backward, f.grad, **{"fwd__" + k: v for k, v in wide.items()}, **ld, workspace_bytes=1 << 62)


@pytest.mark.parametrize("kw", [
    dict(fwd__rows=-1), dict(dy=None), dict(lddy=23), dict(lddx=15), dict(grad_dtype=1), dict(accumulate=1),
    dict(ld_din=15), dict(ld_dout=31), dict(workspace=None), dict(workspace_bytes=16), dict(fwd__act=9),
    dict(fwd__saved=None), dict(dw_down=ADDRESS + 1)])
def test_backward_launcher_refuses(kw):
    f = ffn()
    f.gradients(M(8, 24), dx=M(8, 16), dw_gate=M(32, 16), dw_up=M(32, 16), dw_down=M(24, 32), room=Room())
    if "fwd__saved" in kw and f.args.saved is None:
        pytest.skip("this size recomputes g and u")
    assert refused(nn._lib().b2c_hip_ffn_backward, f.grad, **kw)


class View:
    """What QuantizeRows asks of a tensor: rows x cols bytes, rows ld apart, `first` bytes into a storage of `size`."""

    def __init__(self, rows, cols, ld, first, size):
        self.shape, self.dtype, self._ld, self._first, self._size = (rows, cols), "torch.int8", ld, first, size

    def stride(self, i):
        return 1 if i else self._ld

    def data_ptr(self):
        return ADDRESS + self._first

    def storage_offset(self):
        return self._first

    def untyped_storage(self):
        return self

    def nbytes(self):
        return self._size


@pytest.mark.parametrize("rows,cols,ld,first,size,fits", [
    (4, 5, 5, 0, 20, True), (4, 16, 40, 24, 160, True), (4, 10, 16, 0, 64, True), (4, 10, 16, 6, 64, False), (4, 20, 40, 0, 152, True),
    (4, 20, 40, 0, 140, False), (4, 20, 40, 16, 160, False), (1, 5, 5, 59, 64, True)])
def test_quantize_rows_keeps_to_the_rows_of_a_view(rows, cols, ld, first, size, fits):
    plan = lambda: nn.QuantizeRows(M(rows, cols), View(rows, cols, ld, first, size), nn.Matrix(ADDRESS, rows, 1, 1, nn.F32))  # noqa: E731
    if fits:
        plan()
    else:
        with pytest.raises(ValueError, match="room"):
            plan()


def test_other_launchers_refuse():
    L = nn._lib()
    d = lambda: nn.Dropout(M(4, 5), M(4, 5), 0.1, 1, 2)  # noqa: E731
    for kw in (dict(rows=-1), dict(cols=0), dict(dtype=3), dict(p=1.0), dict(x=None), dict(x=ADDRESS + 1), dict(ldx=4), dict(y=None),
               dict(ldy=4), dict(residual=ADDRESS, ldr=4), dict(rows=1 << 40, cols=1 << 20)):
        assert refused(L.b2c_hip_dropout, d().args, **kw), kw
    q = lambda: nn.QuantizeRows(M(4, 5), M(4, 5, nn.I8), nn.Matrix(ADDRESS, 4, 1, 1, nn.F32))  # noqa: E731
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(dtype=3), dict(x=None), dict(ldx=4), dict(q=None), dict(ldq=4),
               dict(scale=None), dict(scale=ADDRESS + 2)):
        assert refused(L.b2c_hip_quantize_rows, q().args, **kw), kw
    s = lambda n: nn.Matrix(ADDRESS, n, 1, 1, nn.F32)  # noqa: E731
    li = lambda: nn.I8Linear(M(4, 5), M(6, 5, nn.I8), s(6), M(4, 6), room=Room())  # noqa: E731
    for kw in (dict(rows=-1), dict(d_in=0), dict(d_in=131073), dict(d_out=0), dict(dtype=3), dict(x=None), dict(w=None), dict(ldw=4),
               dict(w_scale=None), dict(y=None), dict(ldy=5), dict(workspace=None), dict(workspace_bytes=0)):
        assert refused(L.b2c_hip_i8_linear, li().args, **kw), kw
    bl = lambda: nn.I8FeedForward(M(4, 5), M(7, 5, nn.I8), s(7), M(7, 5, nn.I8), s(7), M(6, 7, nn.I8), s(6), M(4, 6),  # noqa: E731
                                  room=Room())
    for kw in (dict(rows=-1), dict(d_in=0), dict(d_hidden=131073), dict(d_out=0), dict(act=3), dict(w_gate=None), dict(w_up=None),
               dict(w_down=None), dict(s_gate=None), dict(s_up=None), dict(s_down=None), dict(ld_in=4), dict(ld_out=6),
               dict(workspace=None), dict(workspace_bytes=0)):
        assert refused(L.b2c_hip_i8_ffn, bl().args, **kw), kw
    for bad in (lambda: nn.Dropout(M(4, 5), M(4, 6), 0.1, 1, 2), lambda: nn.Dropout(M(4, 5), M(4, 5, nn.F16), 0.1, 1, 2),
                lambda: nn.Dropout(M(4, 5), M(4, 5), 1.0, 1, 2), lambda: nn.Dropout(M(4, 5, nn.I8), M(4, 5, nn.I8), 0.1, 1, 2),
                lambda: nn.I8Linear(M(4, 5), M(6, 5), s(6), M(4, 6), room=Room()),
                lambda: nn.I8Linear(M(4, 5), M(6, 5, nn.I8), s(5), M(4, 6), room=Room()),
                lambda: nn.I8FeedForward(M(4, 5), M(7, 5, nn.I8), s(7), M(8, 5, nn.I8), s(8), M(6, 7, nn.I8), s(6), M(4, 6), room=Room()),
                lambda: nn.QuantizeRows(M(4, 5), M(4, 6, nn.I8), s(4)), lambda: nn.QuantizeRows(M(4, 5), M(4, 5, nn.I8), s(5))):
        with pytest.raises(ValueError):
            bad()


def test_sizes_are_zero_for_bad_arguments_and_grow_with_rows():
    L = nn._lib()
    f = ffn()
    sizes = []
    for rows in (1, 33, 100, 5000):
        f.args.rows = rows
        sizes.append(L.b2c_ffn_workspace_bytes(C.byref(f.args)))
    assert sizes == sorted(sizes) and sizes[0] > 0
    f.args.dtype = 7
    assert L.b2c_ffn_workspace_bytes(C.byref(f.args)) == 0 and L.b2c_ffn_saved_bytes(C.byref(f.args)) == 0


def test_no_rows_is_valid():
    for fn, args in ((nn._lib().b2c_hip_ffn_forward, nn.FfnArgs(rows=0, d_in=4, d_hidden=4, d_out=4, dtype=2)),
                     (nn._lib().b2c_hip_dropout, nn.DropoutArgs(rows=0, cols=4, dtype=2)),
                     (nn._lib().b2c_hip_i8_linear, nn.I8LinearArgs(rows=0, d_in=4, d_out=4, dtype=2)),
                     (nn._lib().b2c_hip_i8_ffn, nn.I8FfnArgs(rows=0, d_in=4, d_hidden=4, d_out=4, dtype=2)),
                     (nn._lib().b2c_hip_quantize_rows, nn.QuantizeArgs(rows=0, cols=4, dtype=2))):
        assert fn(C.byref(args), None) == 0
