"""The norms between blocks, 4-bit weights and experts without a GPU: what their plans and launchers refuse, and the tests' own restatement
of them against differences."""
import ctypes as C

import numpy as np
import pytest
import torch

from b2ctrain_amd import _native, nn
from tests import dense_util as U
from tests import more_util as V
from tests.test_dense_host import ADDRESS, M, Room, refused

F32, F16, BF16 = nn.F32, nn.F16, nn.BF16


def row(n, dtype=BF16, ptr=ADDRESS):
    return nn.Matrix(ptr, 1, n, n, dtype)


# ---- the restatement ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
@pytest.mark.parametrize("post", [False, True])
def test_block_norm_gradients_against_differences(kind, act, post):
    """Central differences in 64 bits: off by the step squared and by rounding / step."""
    g = np.random.default_rng(4)
    rows, d, per = 7, 6, 3
    v = dict(x=g.standard_normal((rows, d)), r=g.standard_normal((rows, d)), gate=g.standard_normal((3, d)), w_post=1 + 0.2 * g.standard_normal(d),
             w_pre=1 + 0.2 * g.standard_normal(d))
    dy, dn = g.standard_normal((rows, d)), g.standard_normal((rows, d))
    if not post:
        v["w_post"] = None
    call = lambda **kw: V.block_norm(F32, F32, per=per, act=act, post=post, kind=kind, eps=1e-3, scale=0.5, **v, **kw)  # noqa: E731
    grads, h = call(dy=dy, dn=dn), 1e-5
    for key, name in (("x", "dx"), ("r", "dresidual"), ("gate", "dgate"), ("w_post", "dw_post"), ("w_pre", "dw_pre")):
        if v[key] is None:
            continue
        for idx in zip(*(g.integers(0, n, 12) for n in v[key].shape)):
            keep, side = v[key][idx], []
            for s in (h, -h):
                v[key][idx] = keep + s
                out = call()
                side.append((out["y"][0] * dy).sum() + (out["n"][0] * dn).sum())
            v[key][idx] = keep
            want = grads[name][0][idx]
            assert abs((side[0] - side[1]) / (2 * h) - want) < 1e-6 * (1 + abs(want)), (key, idx)


def test_quantised_groups_stand_for_what_they_hold():
    """Codes stay within half a step of the values, and the step is the group's largest magnitude over 7 or its reach over 15."""
    g = np.random.default_rng(1)
    x = g.standard_normal((9, 70)).astype(np.float32)
    for zeros in (False, True):
        code, stored, zero, values = V.quantised4(x, 32, zeros, BF16)
        s = np.repeat(U.value(stored, BF16), 32, axis=1)[:, :70]
        assert (abs(values - x) <= (0.5 + (1.0 if zeros else 7.5 * 2.0 ** -8)) * s).all() and code.max() <= 15
        assert np.array_equal(V.packed(code)[:, 0] & 15, code[:, 0]) and np.array_equal(V.packed(code)[:, -1] >> 4, code[:, -1])


def test_experts_of_one_are_a_block():
    g = np.random.default_rng(2)
    x, wr, wg, wu, wd = (g.standard_normal(s) for s in ((4, 6), (1, 6), (9, 6), (9, 6), (5, 9)))
    assert np.allclose(V.experts(x, wr, wg, wu, wd, 1, "gelu", BF16)[2], U.block(x, wg, wu, wd, "gelu"), rtol=1e-12)


# ---- plans -------------------------------------------------------------------------------------------------

def norm(**kw):
    a = dict(x=M(8, 16), residual=M(8, 16), y=M(8, 16), n=M(8, 16), gate=M(4, 16), rows_per_gate=2, post=True, w_post=row(16), w_pre=row(16))
    a.update(kw)
    return nn.BlockNorm(**{k: v for k, v in a.items() if v is not None})


@pytest.mark.parametrize("kw", [
    dict(x=M(8, 17)), dict(x=M(8, 16, F16)), dict(x=M(8, 16, nn.I8)), dict(residual=M(7, 16)), dict(y=M(8, 15)), dict(n=M(9, 16)),
    dict(gate=M(3, 16)), dict(gate=M(4, 15)), dict(rows_per_gate=None), dict(rows_per_gate=0), dict(rows_per_gate=1), dict(gate=None),
    dict(gate_act="tanh"), dict(kind="batch"), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(post=False),
    dict(w_post=row(15)), dict(w_pre=row(16, F32)), dict(w_pre=row(16, F16)), dict(w_post=row(16, ptr=0)), dict(n=None), dict(x=None),
    dict(x=None, gate=None, rows_per_gate=None, post=False, w_post=None), dict(y=None, n=None, w_pre=None), dict(x=3),
    dict(x=M(8, 16, ld=15)), dict(w_pre=torch.ones(16, dtype=torch.bfloat16))])
def test_block_norm_plan_refuses(kw):
    norm()
    with pytest.raises(ValueError):
        norm(**kw)


def test_block_norm_takes_one_gate_row_for_all_or_one_for_each():
    for rows, per in ((1, 8), (8, 1)):
        assert norm(gate=M(rows, 16), rows_per_gate=None).args.rows_per_gate == per
    with pytest.raises(ValueError, match="columns"):
        nn.BlockNorm(residual=M(4, 16385), n=M(4, 16385))
    assert nn.BlockNorm(residual=M(4, 16384), n=M(4, 16384)).args.cols == 16384


@pytest.mark.parametrize("kw", [
    dict(dy=None, dn=None), dict(dy=M(8, 15)), dict(dn=M(7, 16)), dict(dx=M(8, 16, F32)), dict(dresidual=M(8, 17)), dict(dgate=M(8, 16)),
    dict(dw_post=row(15)), dict(dw_pre=row(16, F16)), dict(dw_post=row(16), dw_pre=row(16, F32)), dict(dw_pre=row(16), accumulate=True),
    dict(dn=None, dw_pre=row(16)), dict(dw_post=row(16), room=None)])
def test_block_norm_gradient_plan_refuses(kw):
    a = dict(dy=M(8, 16), dn=M(8, 16), room=Room())
    norm().gradients(**a, dgate=M(4, 16), dw_post=row(16), dw_pre=row(16))
    with pytest.raises(ValueError):
        norm().gradients(**{**a, **kw})
    for form, wanted in ((dict(gate=None, rows_per_gate=None), dict(dgate=M(4, 16))), (dict(post=False, w_post=None), dict(dw_post=row(16)))):
        with pytest.raises(ValueError, match="what was not given"):
            norm(**form).gradients(**a, **wanted)
    with pytest.raises(ValueError, match="gradients"):
        norm().backward()


def pack(**kw):
    return nn.QuantizeGroups(**{**dict(x=M(4, 70), q=M(4, 35, nn.U8), scale=M(4, 3), group=32, zero=M(4, 3, nn.U8), values=M(4, 70)), **kw})


@pytest.mark.parametrize("kw", [
    dict(x=M(4, 71)), dict(x=M(4, 70, nn.I8)), dict(q=M(4, 34, nn.U8)), dict(q=M(4, 35, nn.I8)), dict(q=M(5, 35, nn.U8)), dict(scale=M(4, 2)),
    dict(scale=M(4, 3, F32)), dict(group=16), dict(group=48), dict(group=0), dict(group=64), dict(zero=M(4, 2, nn.U8)), dict(zero=M(4, 3)),
    dict(values=M(4, 70, F32))])
def test_quantise_plan_refuses(kw):
    pack()
    with pytest.raises(ValueError):
        pack(**kw)


def q4(**kw):
    return nn.Q4Linear(**{**dict(x=M(4, 70), w=M(9, 35, nn.U8), scale=M(9, 3), y=M(4, 9), group=32, zero=M(9, 3, nn.U8), room=Room()), **kw})


@pytest.mark.parametrize("kw", [
    dict(x=M(4, 70, F32)), dict(x=M(4, 71)), dict(w=M(9, 35, nn.I8)), dict(w=M(9, 36, nn.U8)), dict(scale=M(9, 3, F16)), dict(scale=M(8, 3)),
    dict(zero=M(9, 4, nn.U8)), dict(y=M(4, 8)), dict(y=M(4, 9, F32)), dict(group=100), dict(w=M(9, 35, nn.U8, ld=(1 << 25) + 1)),
    dict(x=M(3000, 70), y=M(3000, 9), room=None)])
def test_q4_linear_plan_refuses(kw):
    q4()
    with pytest.raises(ValueError):
        q4(**kw)


def experts(**kw):
    a = dict(x=M(4, 10), w_router=M(3, 10), w_gate=M(21, 10), w_up=M(21, 10), w_down=M(18, 7), y=M(4, 6), top_k=2, residual=M(4, 6),
             index=M(4, 2, nn.I32), weight=M(4, 2, F32), room=Room())
    return nn.Experts(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(x=M(4, 10, F32)), dict(w_router=M(3, 9)), dict(w_router=M(4, 10)), dict(w_router=M(3, 10, F16)), dict(w_gate=M(20, 10)), dict(w_up=M(24, 10)),
    dict(w_up=M(21, 10, ld=12)), dict(w_down=M(17, 7)), dict(w_down=M(18, 8)), dict(y=M(4, 7)), dict(y=M(3, 6)), dict(top_k=0), dict(top_k=4),
    dict(act="tanh"), dict(residual=M(4, 5)), dict(index=M(4, 2, F32)), dict(index=M(4, 3, nn.I32)), dict(weight=M(4, 2)), dict(room=None),
    dict(w_down=M(18, 7, ld=1 << 26)), dict(w_router=M(1025, 10), w_gate=M(1025, 10), w_up=M(1025, 10), w_down=M(6150, 1)),
    dict(w_router=M(65, 10), w_gate=M(65, 10), w_up=M(65, 10), w_down=M(390, 1), top_k=65, index=None, weight=None)])
def test_experts_plan_refuses(kw):
    experts()
    with pytest.raises(ValueError):
        experts(**kw)


# ---- launchers ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=16385), dict(dtype=3), dict(dtype=-1), dict(w_dtype=1), dict(kind=2), dict(kind=-1),
    dict(gate_act=2), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(x=ADDRESS + 1), dict(ldx=15),
    dict(residual=ADDRESS + 1), dict(ldr=15), dict(gate=ADDRESS + 1), dict(ldg=15), dict(rows_per_gate=0), dict(post=0), dict(w_post=ADDRESS + 1),
    dict(w_pre=ADDRESS + 1), dict(y=ADDRESS + 1), dict(ldy=15), dict(n=ADDRESS + 1), dict(ldn=15), dict(y=None, n=None)])
def test_block_norm_launcher_refuses(kw):
    assert refused(nn._lib().b2c_hip_block_norm, norm().args, **kw)


@pytest.mark.parametrize("kw", [
    dict(fwd__rows=-1), dict(fwd__cols=16385), dict(fwd__x=None), dict(dy=None, dn=None, dw_pre=None), dict(dn=None), dict(lddy=15), dict(lddn=15),
    dict(lddx=15), dict(lddr=15), dict(lddg=15), dict(dx=ADDRESS + 1), dict(grad_dtype=1), dict(grad_dtype=7), dict(accumulate=1), dict(fwd__gate=None),
    dict(dw_post=ADDRESS + 1), dict(dw_pre=ADDRESS + 1), dict(workspace=None), dict(workspace=ADDRESS + 8), dict(workspace_bytes=16),
    dict(fwd__post=0, fwd__w_post=None)])
def test_block_norm_gradient_launcher_refuses(kw):
    p = norm()
    p.gradients(dy=M(8, 16), dn=M(8, 16), dx=M(8, 16), dresidual=M(8, 16), dgate=M(4, 16), dw_post=row(16), dw_pre=row(16), room=Room())
    assert refused(nn._lib().b2c_hip_block_norm_backward, p.grad, **kw)


def test_other_launchers_refuse():
    L = nn._lib()
    for kw in (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=(1 << 20) + 1), dict(group=33), dict(group=512), dict(dtype=3), dict(scale_dtype=0),
               dict(x=None), dict(x=ADDRESS + 1), dict(ldx=69), dict(q=None), dict(ldq=34), dict(scale=None), dict(scale=ADDRESS + 1), dict(lds=2),
               dict(ldz=2), dict(values=ADDRESS + 1), dict(ldv=69)):
        assert refused(L.b2c_hip_quantize4, pack().args, **kw), kw
    for kw in (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(d_in=0), dict(d_in=(1 << 20) + 1), dict(d_out=0), dict(d_out=(1 << 20) + 1), dict(group=7),
               dict(dtype=0), dict(dtype=3), dict(x=None), dict(x=ADDRESS + 1), dict(ldx=69), dict(w=None), dict(ldw=34), dict(ldw=(1 << 25) + 1),
               dict(scale=None), dict(scale=ADDRESS + 1), dict(lds=2), dict(lds=1 << 26), dict(ldz=2), dict(ldz=1 << 26), dict(y=None), dict(ldy=8)):
        assert refused(L.b2c_hip_q4_linear, q4().args, **kw), kw
    for kw in (dict(workspace=None), dict(workspace=ADDRESS + 8), dict(workspace_bytes=16)):
        assert refused(L.b2c_hip_q4_linear, q4(x=M(3000, 70), y=M(3000, 9)).args, **kw), kw
    for kw in (dict(rows=-1), dict(rows=(1 << 20) + 1), dict(d_in=0), dict(d_hidden=0), dict(d_out=0), dict(d_out=(1 << 20) + 1), dict(experts=0),
               dict(experts=1025), dict(top_k=0), dict(top_k=4), dict(dtype=0), dict(act=3), dict(x=None), dict(ldx=9), dict(w_router=None),
               dict(ld_router=9), dict(w_gate=None), dict(w_up=None), dict(w_up=ADDRESS + 1), dict(ld_in=9), dict(ld_in=1 << 26), dict(w_down=None),
               dict(ld_out=6), dict(ld_out=1 << 26), dict(ldr=5), dict(y=None), dict(ldy=5), dict(index=ADDRESS + 2), dict(ldi=1),
               dict(weight=ADDRESS + 2), dict(ldw=1), dict(workspace=None), dict(workspace=ADDRESS + 8), dict(workspace_bytes=16),
               dict(experts=1024, top_k=2, d_hidden=1 << 20, d_out=1 << 20, ld_out=1 << 20, workspace_bytes=1 << 40),
               dict(experts=1024, d_hidden=1 << 21)):
        assert refused(L.b2c_hip_experts, experts().args, **kw), kw


def test_no_rows_is_valid_and_needs_no_workspace():
    L = nn._lib()
    for fn, room, args in (
            (L.b2c_hip_block_norm, None, nn.BlockNormArgs(rows=0, cols=4, dtype=2, w_dtype=2, x=ADDRESS)),
            (L.b2c_hip_quantize4, None, nn.Quantize4Args(rows=0, cols=4, group=32, dtype=2, scale_dtype=2)),
            (L.b2c_hip_q4_linear, L.b2c_q4_linear_workspace_bytes, nn.Q4LinearArgs(rows=0, d_in=4, d_out=4, group=32, dtype=2)),
            (L.b2c_hip_experts, L.b2c_experts_workspace_bytes, nn.ExpertsArgs(rows=0, d_in=4, d_hidden=4, d_out=4, experts=2, top_k=1, dtype=2))):
        assert fn(C.byref(args), None) == 0 and (room is None or room(C.byref(args)) == 0)
        assert fn(None, None) == 1


def test_workspaces_grow_with_rows_and_end_at_a_lot():
    sizes = [experts(x=M(n, 10), y=M(n, 6), residual=None, index=None, weight=None).args.workspace_bytes for n in (2, 40, 512, 513, 100000)]
    assert sizes == sorted(sizes) and sizes[2] == sizes[3] == sizes[4]
    sizes = [q4(x=M(n, 70), y=M(n, 9)).args.workspace_bytes for n in (1, 32, 600, 5000)]
    assert sizes[0] == sizes[1] == 0 < sizes[2] <= sizes[3]


@pytest.mark.parametrize("entry,args,handle", [("b2c_block_norm", nn.BlockNormArgs, False), ("b2c_block_norm_backward", nn.BlockNormGradArgs, True),
                                               ("b2c_quantize4", nn.Quantize4Args, False), ("b2c_q4_linear", nn.Q4LinearArgs, True),
                                               ("b2c_experts", nn.ExpertsArgs, True)])
def test_a_null_handle_or_argument_is_an_error(entry, args, handle):
    L, p = _native.lib(), C.c_void_p
    fn = getattr(L, entry)
    fn.argtypes = [p, p, p] if handle else [p, p]
    L.b2c_dense_create.restype, L.b2c_dense_destroy.argtypes = p, [p]
    d, some = L.b2c_dense_create(), args(rows=-1) if args is not nn.BlockNormGradArgs else args()
    try:
        for h, a in ((None, C.addressof(some)), (d, None), (None, None)) if handle else ((None, None),):
            assert fn(*([h] if handle else []), a, None) != 0 and b"null" in L.b2c_last_error()
        if args is not nn.BlockNormGradArgs:
            assert fn(*([d] if handle else []), C.addressof(some), None) != 0 and b"invalid arguments" in L.b2c_last_error()
    finally:
        L.b2c_dense_destroy(d)
