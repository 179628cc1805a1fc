"""Dense operators of a learned head over splats or tokens: the gated feed-forward block with its gradients, dropout, the norms
between two blocks with their gradients, products in 8-bit integers and with 4-bit weights, and a mixture of experts for a few
tokens (include/b2c_kernels.h, "dense operators").

An operator is planned once for its matrices and then run on a HIP stream as often as wanted: the plan holds the
launcher's argument struct, and allocates nothing but through `room`, a function that the caller gives (bytes -> an
object with `data_ptr()` or `ptr`; in a torch program ``lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")``). A matrix is
a two-dimensional torch tensor whose columns lie next to each other, or a ``Matrix`` over any device pointer. Plans keep
what they point at alive. Streams are the integer handle of a HIP stream (0: the default stream), and the caller orders
work on different streams, as for every launcher.

    f = nn.FeedForward(x, w_gate, w_up, w_down, y, p=0.1, seed=7, train=True, room=room)
    f.gradients(dy, dx=dx, dw_gate=dwg, dw_up=dwu, dw_down=dwd, room=room)
    for step in range(n):
        f.set_stream_id(step)          # another mask each step
        f.forward(stream)
        ...                            # dy from y
        f.backward(stream)

A wrong argument raises ValueError before anything is launched; a launch that fails raises RuntimeError.
"""
from __future__ import annotations

import ctypes as C

from b2ctrain_amd import _native

F32, F16, BF16 = 0, 1, 2
I8, U8, I32 = 3, 4, 5  # of a Matrix only
SIZES = {F32: 4, F16: 2, BF16: 2, I8: 1, U8: 1, I32: 4}
NAMES = {"float32": F32, "float16": F16, "bfloat16": BF16, "int8": I8, "uint8": U8, "int32": I32}
ACTS = {"silu": 0, "gelu": 1, "relu": 2}
NORMS = {"rms": 0, "layer": 1}
GATES = {"none": 0, "sigmoid": 1}
GROUPS = (32, 64, 128, 256)

_i64, _int, _f32, _u64, _ptr, _size = C.c_int64, C.c_int, C.c_float, C.c_uint64, C.c_void_p, C.c_size_t


class DropoutArgs(C.Structure):
    _fields_ = [("rows", _i64), ("cols", _i64), ("dtype", _int), ("p", _f32), ("seed", _u64), ("stream", _u64), ("x", _ptr),
                ("ldx", _i64), ("residual", _ptr), ("ldr", _i64), ("y", _ptr), ("ldy", _i64)]


class FfnArgs(C.Structure):
    _fields_ = [("rows", _i64), ("d_in", _int), ("d_hidden", _int), ("d_out", _int), ("dtype", _int), ("act", _int),
                ("p", _f32), ("seed", _u64), ("stream", _u64), ("x", _ptr), ("ldx", _i64), ("w_gate", _ptr), ("w_up", _ptr),
                ("ld_in", _i64), ("w_down", _ptr), ("ld_out", _i64), ("residual", _ptr), ("ldr", _i64), ("y", _ptr),
                ("ldy", _i64), ("saved", _ptr), ("workspace", _ptr), ("workspace_bytes", _size)]


class FfnGradArgs(C.Structure):
    _fields_ = [("fwd", FfnArgs), ("dy", _ptr), ("lddy", _i64), ("dx", _ptr), ("lddx", _i64), ("grad_dtype", _int),
                ("accumulate", _int), ("dw_gate", _ptr), ("dw_up", _ptr), ("ld_din", _i64), ("dw_down", _ptr),
                ("ld_dout", _i64), ("workspace", _ptr), ("workspace_bytes", _size)]


class QuantizeArgs(C.Structure):
    _fields_ = [("rows", _i64), ("cols", _i64), ("dtype", _int), ("x", _ptr), ("ldx", _i64), ("q", _ptr), ("ldq", _i64),
                ("scale", _ptr)]


class I8LinearArgs(C.Structure):
    _fields_ = [("rows", _i64), ("d_in", _int), ("d_out", _int), ("dtype", _int), ("x", _ptr), ("ldx", _i64), ("w", _ptr),
                ("ldw", _i64), ("w_scale", _ptr), ("y", _ptr), ("ldy", _i64), ("workspace", _ptr),
                ("workspace_bytes", _size)]


class I8FfnArgs(C.Structure):
    _fields_ = [("rows", _i64), ("d_in", _int), ("d_hidden", _int), ("d_out", _int), ("dtype", _int), ("act", _int),
                ("x", _ptr), ("ldx", _i64), ("w_gate", _ptr), ("w_up", _ptr), ("ld_in", _i64), ("s_gate", _ptr),
                ("s_up", _ptr), ("w_down", _ptr), ("ld_out", _i64), ("s_down", _ptr), ("y", _ptr), ("ldy", _i64),
                ("workspace", _ptr), ("workspace_bytes", _size)]


class BlockNormArgs(C.Structure):
    _fields_ = [("rows", _i64), ("cols", _int), ("dtype", _int), ("w_dtype", _int), ("kind", _int), ("post", _int), ("gate_act", _int),
                ("eps", _f32), ("scale", _f32), ("x", _ptr), ("ldx", _i64), ("residual", _ptr), ("ldr", _i64), ("gate", _ptr),
                ("ldg", _i64), ("rows_per_gate", _i64), ("w_post", _ptr), ("w_pre", _ptr), ("y", _ptr), ("ldy", _i64), ("n", _ptr),
                ("ldn", _i64)]


class BlockNormGradArgs(C.Structure):
    _fields_ = [("fwd", BlockNormArgs), ("dy", _ptr), ("lddy", _i64), ("dn", _ptr), ("lddn", _i64), ("dx", _ptr), ("lddx", _i64),
                ("dresidual", _ptr), ("lddr", _i64), ("dgate", _ptr), ("lddg", _i64), ("grad_dtype", _int), ("accumulate", _int),
                ("dw_post", _ptr), ("dw_pre", _ptr), ("workspace", _ptr), ("workspace_bytes", _size)]


class Quantize4Args(C.Structure):
    _fields_ = [("rows", _i64), ("cols", _int), ("group", _int), ("dtype", _int), ("scale_dtype", _int), ("x", _ptr), ("ldx", _i64),
                ("q", _ptr), ("ldq", _i64), ("scale", _ptr), ("lds", _i64), ("zero", _ptr), ("ldz", _i64), ("values", _ptr),
                ("ldv", _i64)]


class Q4LinearArgs(C.Structure):
    _fields_ = [("rows", _i64), ("d_in", _int), ("d_out", _int), ("group", _int), ("dtype", _int), ("x", _ptr), ("ldx", _i64),
                ("w", _ptr), ("ldw", _i64), ("scale", _ptr), ("lds", _i64), ("zero", _ptr), ("ldz", _i64), ("y", _ptr), ("ldy", _i64),
                ("workspace", _ptr), ("workspace_bytes", _size)]


class ExpertsArgs(C.Structure):
    _fields_ = [("rows", _i64), ("d_in", _int), ("d_hidden", _int), ("d_out", _int), ("experts", _int), ("top_k", _int),
                ("dtype", _int), ("act", _int), ("normalize", _int), ("x", _ptr), ("ldx", _i64), ("w_router", _ptr),
                ("ld_router", _i64), ("w_gate", _ptr), ("w_up", _ptr), ("ld_in", _i64), ("w_down", _ptr), ("ld_out", _i64),
                ("residual", _ptr), ("ldr", _i64), ("y", _ptr), ("ldy", _i64), ("index", _ptr), ("ldi", _i64), ("weight", _ptr),
                ("ldw", _i64), ("workspace", _ptr), ("workspace_bytes", _size)]


_bound = False


def _lib():
    global _bound
    L = _native.lib()
    if not _bound:
        for name, args in (("dropout", DropoutArgs), ("ffn_forward", FfnArgs), ("ffn_backward", FfnGradArgs),
                           ("quantize_rows", QuantizeArgs), ("i8_linear", I8LinearArgs), ("i8_ffn", I8FfnArgs),
                           ("block_norm", BlockNormArgs), ("block_norm_backward", BlockNormGradArgs), ("quantize4", Quantize4Args),
                           ("q4_linear", Q4LinearArgs), ("experts", ExpertsArgs)):
            fn = getattr(L, "b2c_hip_" + name)
            fn.argtypes, fn.restype = [C.POINTER(args), _ptr], _int
        for name, args in (("b2c_ffn_saved_bytes", FfnArgs), ("b2c_ffn_workspace_bytes", FfnArgs),
                           ("b2c_ffn_grad_workspace_bytes", FfnGradArgs), ("b2c_i8_linear_workspace_bytes", I8LinearArgs),
                           ("b2c_i8_ffn_workspace_bytes", I8FfnArgs),
                           ("b2c_block_norm_grad_workspace_bytes", BlockNormGradArgs),
                           ("b2c_q4_linear_workspace_bytes", Q4LinearArgs), ("b2c_experts_workspace_bytes", ExpertsArgs)):
            fn = getattr(L, name)
            fn.argtypes, fn.restype = [C.POINTER(args)], _size
        _bound = True
    return L


class Matrix:
    """rows x cols values at a device pointer, rows `ld` values apart. `keep`: what owns the memory."""

    def __init__(self, ptr, rows, cols, ld, dtype, keep=None):
        self.ptr, self.rows, self.cols, self.ld, self.dtype, self.keep = ptr, rows, cols, ld, dtype, keep


def matrix(what, name, rows=None, cols=None, dtype=None):
    """`what` as a Matrix, checked against the wanted shape and type."""
    m = what
    if not isinstance(m, Matrix):
        try:
            if len(m.shape) != 2:
                raise ValueError(f"{name}: a matrix is wanted, got {len(m.shape)} dimensions")
            r, c = int(m.shape[0]), int(m.shape[1])
            kind = NAMES.get(str(m.dtype).replace("torch.", ""))
            if getattr(m, "is_cuda", True) is False:
                raise ValueError(f"{name}: is not on the GPU")
            if c > 1 and m.stride(1) != 1:
                raise ValueError(f"{name}: columns have to lie next to each other")
            ld = int(m.stride(0)) if r > 1 else max(c, 1)
            m = Matrix(m.data_ptr(), r, c, ld, kind, keep=what)
        except AttributeError:
            raise ValueError(f"{name}: a matrix is wanted, got {type(what).__name__}") from None
    if m.dtype is None or (dtype is not None and m.dtype != dtype):
        raise ValueError(f"{name}: has another type than wanted")
    if (rows is not None and m.rows != rows) or (cols is not None and m.cols != cols):
        raise ValueError(f"{name}: is {m.rows} x {m.cols}, wanted {'?' if rows is None else rows} x {'?' if cols is None else cols}")
    if m.cols < 1:
        raise ValueError(f"{name}: has no columns")
    if m.rows > 1 and m.ld < m.cols:
        raise ValueError(f"{name}: rows overlap")
    if m.rows and not m.ptr:
        raise ValueError(f"{name}: a null pointer")
    return m


def _vector(what, name, n):
    """The pointer of n single-precision values on the GPU."""
    if isinstance(what, Matrix):
        m, fits = what, what.rows * what.cols == n and (what.rows <= 1 or what.ld == what.cols)
    else:
        try:
            fits = tuple(what.shape) == (n,) and (n <= 1 or what.stride(0) == 1)
            if getattr(what, "is_cuda", True) is False:
                raise ValueError(f"{name}: is not on the GPU")
            m = Matrix(what.data_ptr(), n, 1, 1, NAMES.get(str(what.dtype).replace("torch.", "")), keep=what)
        except AttributeError:
            raise ValueError(f"{name}: {n} single-precision values are wanted, got {type(what).__name__}") from None
    if m.dtype != F32 or not fits:
        raise ValueError(f"{name}: {n} single-precision values next to each other are wanted")
    if n and not m.ptr:
        raise ValueError(f"{name}: a null pointer")
    return m.ptr


def _floating(m, name, types=(F32, F16, BF16)):
    if m.dtype not in types:
        raise ValueError(f"{name}: its type is not supported here")
    return m


def _chance(p):
    p = float(p)
    if not 0.0 <= p < 1.0 or int(C.c_float(p).value * 65536.0 + 0.5) >= 65536:
        raise ValueError(f"dropout probability {p}: wanted 0 <= p < 1, at most 65535 / 65536")
    return p


def _act(act):
    if act not in ACTS:
        raise ValueError(f"activation {act!r}: wanted one of {', '.join(ACTS)}")
    return ACTS[act]


def _check(rc, what):
    if rc == 1:
        raise ValueError(f"{what}: invalid arguments")
    if rc != 0:
        raise RuntimeError(f"{what}: HIP error {rc}")


def _get_room(room, n, what):
    if n == 0:
        return None, None
    if room is None:
        raise ValueError(f"{what}: needs {n} bytes of workspace: give `room`")
    b = room(n)
    at = b.data_ptr() if hasattr(b, "data_ptr") else getattr(b, "ptr", None)
    if not at or getattr(b, "is_cuda", True) is False or getattr(b, "nbytes", n) < n:
        raise ValueError(f"{what}: `room` has to give {n} bytes of workspace on the GPU")
    return b, at


class Dropout:
    """y = residual + dropout(x); b2c_hip_dropout. y may be x or residual. The gradient of x is a Dropout of y's
    gradient with the same p, seed and stream_id."""

    def __init__(self, x, y, p, seed, stream_id, residual=None):
        x = _floating(matrix(x, "x"), "x")
        y = matrix(y, "y", x.rows, x.cols, x.dtype)
        r = matrix(residual, "residual", x.rows, x.cols, x.dtype) if residual is not None else None
        self._keep = (x, y, r)
        self.args = DropoutArgs(rows=x.rows, cols=x.cols, dtype=x.dtype, p=_chance(p), seed=seed % (1 << 64),
                                stream=stream_id % (1 << 64), x=x.ptr, ldx=x.ld, residual=r.ptr if r else None,
                                ldr=r.ld if r else 0, y=y.ptr, ldy=y.ld)
        self._fn, self._ref = _lib().b2c_hip_dropout, C.byref(self.args)

    def set_stream_id(self, stream_id):
        self.args.stream = stream_id % (1 << 64)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "dropout")


class FeedForward:
    """y = residual + dropout((act(x w_gate') * (x w_up')) w_down'), and its gradients; b2c_hip_ffn_forward and
    b2c_hip_ffn_backward. Weights are [outputs, inputs]. y may be residual. `train`: keep what backward() needs."""

    def __init__(self, x, w_gate, w_up, w_down, y, act="silu", residual=None, p=0.0, seed=0, stream_id=0, train=False, room=None):
        L = _lib()
        x = _floating(matrix(x, "x"), "x", (F16, BF16))
        g = matrix(w_gate, "w_gate", None, x.cols, x.dtype)
        u = matrix(w_up, "w_up", g.rows, x.cols, x.dtype)
        d = matrix(w_down, "w_down", None, g.rows, x.dtype)
        if g.rows < 1 or d.rows < 1:
            raise ValueError("feed-forward: a weight has no rows")
        if g.ld != u.ld:
            raise ValueError("feed-forward: w_gate and w_up have different distances between rows")
        y = matrix(y, "y", x.rows, d.rows, x.dtype)
        r = matrix(residual, "residual", x.rows, d.rows, x.dtype) if residual is not None else None
        self.train, self.shape = bool(train), (x.rows, x.cols, g.rows, d.rows)
        self._keep, self._type = [x, g, u, d, y, r], x.dtype
        a = self.args = FfnArgs(rows=x.rows, d_in=x.cols, d_hidden=g.rows, d_out=d.rows, dtype=x.dtype, act=_act(act),
                                p=_chance(p), seed=seed % (1 << 64), stream=stream_id % (1 << 64), x=x.ptr, ldx=x.ld,
                                w_gate=g.ptr, w_up=u.ptr, ld_in=g.ld, w_down=d.ptr, ld_out=d.ld,
                                residual=r.ptr if r else None, ldr=r.ld if r else 0, y=y.ptr, ldy=y.ld)
        self._ref, self._fwd, self._bwd = C.byref(a), L.b2c_hip_ffn_forward, L.b2c_hip_ffn_backward
        if self.train:
            b, a.saved = _get_room(room, L.b2c_ffn_saved_bytes(self._ref), "feed-forward")
            self._keep.append(b)
        a.workspace_bytes = L.b2c_ffn_workspace_bytes(self._ref)
        b, a.workspace = _get_room(room, a.workspace_bytes, "feed-forward")
        self._keep.append(b)
        self.grad = None

    def gradients(self, dy, dx=None, dw_gate=None, dw_up=None, dw_down=None, accumulate=False, room=None):
        """Plans backward(): dy in, and whichever outputs are given. Weight gradients are of the weights' type, or in
        single precision, where `accumulate` adds to what they hold."""
        if not self.train:
            raise ValueError("feed-forward: planned without train=True")
        m, di, f, do = self.shape
        t = self._type
        dy = matrix(dy, "dy", m, do, t)
        dx = matrix(dx, "dx", m, di, t) if dx is not None else None
        ws = [matrix(w, n, r, c) if w is not None else None
              for w, n, r, c in ((dw_gate, "dw_gate", f, di), (dw_up, "dw_up", f, di), (dw_down, "dw_down", do, f))]
        types = {w.dtype for w in ws if w}
        if len(types) > 1 or not types <= {t, F32}:
            raise ValueError("feed-forward: weight gradients are all of the weights' type, or all in single precision")
        if ws[0] and ws[1] and ws[0].ld != ws[1].ld:
            raise ValueError("feed-forward: dw_gate and dw_up have different distances between rows")
        kind = types.pop() if types else F32
        if accumulate and kind != F32:
            raise ValueError("feed-forward: gradients accumulate in single precision only")
        g = self.grad = FfnGradArgs(fwd=self.args, dy=dy.ptr, lddy=dy.ld, dx=dx.ptr if dx else None, lddx=dx.ld if dx else 0,
                                    grad_dtype=kind, accumulate=int(bool(accumulate)))
        for w, field in zip(ws, ("dw_gate", "dw_up", "dw_down")):
            setattr(g, field, w.ptr if w else None)
        g.ld_din = next((w.ld for w in ws[:2] if w), 0)
        g.ld_dout = ws[2].ld if ws[2] else 0
        self._gref = C.byref(g)
        g.workspace_bytes = _lib().b2c_ffn_grad_workspace_bytes(self._gref)
        b, g.workspace = _get_room(room, g.workspace_bytes, "feed-forward gradients")
        self._gkeep = [dy, dx, ws, b]

    def set_stream_id(self, stream_id):
        self.args.stream = stream_id % (1 << 64)
        if self.grad is not None:
            self.grad.fwd.stream = self.args.stream

    def forward(self, stream=0):
        _check(self._fwd(self._ref, stream), "feed-forward")

    def backward(self, stream=0):
        if self.grad is None:
            raise ValueError("feed-forward: plan gradients() first")
        _check(self._bwd(self._gref, stream), "feed-forward gradients")


class QuantizeRows:
    """q, scale = x in 8 bits by rows; b2c_hip_quantize_rows. For weights [outputs, inputs], rows are channels. Where q's rows are
    further apart than wide, the columns between them become 0 up to the next multiple of 16: a view has to leave room for
    them in its own rows."""

    def __init__(self, x, q, scale):
        x = _floating(matrix(x, "x"), "x")
        q = matrix(q, "q", x.rows, x.cols, I8)
        if hasattr(q.keep, "untyped_storage"):
            wide, first = min(-(-q.cols // 16) * 16, q.ld), q.keep.storage_offset()
            ends = first + (q.rows - 1) * q.ld + wide
            if q.rows and wide > q.cols and (first % q.ld + wide > q.ld or ends > q.keep.untyped_storage().nbytes()):
                raise ValueError("q: its last columns have no room for the zeros up to the next multiple of 16")
        self._keep = (x, q, scale)
        self.args = QuantizeArgs(rows=x.rows, cols=x.cols, dtype=x.dtype, x=x.ptr, ldx=x.ld, q=q.ptr, ldq=q.ld,
                                 scale=_vector(scale, "scale", x.rows))
        self._fn, self._ref = _lib().b2c_hip_quantize_rows, C.byref(self.args)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "quantize_rows")


class I8Linear:
    """y = x w' with x quantised by rows within the call and w held in 8 bits with a scale for each output;
    b2c_hip_i8_linear."""

    def __init__(self, x, w, w_scale, y, room=None):
        L = _lib()
        x = _floating(matrix(x, "x"), "x")
        w = matrix(w, "w", None, x.cols, I8)
        y = matrix(y, "y", x.rows, w.rows, x.dtype)
        a = self.args = I8LinearArgs(rows=x.rows, d_in=x.cols, d_out=w.rows, dtype=x.dtype, x=x.ptr, ldx=x.ld, w=w.ptr,
                                     ldw=w.ld, w_scale=_vector(w_scale, "w_scale", w.rows), y=y.ptr, ldy=y.ld)
        self._fn, self._ref = L.b2c_hip_i8_linear, C.byref(a)
        a.workspace_bytes = L.b2c_i8_linear_workspace_bytes(self._ref)
        b, a.workspace = _get_room(room, a.workspace_bytes, "i8_linear")
        self._keep = (x, w, w_scale, y, b)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "i8_linear")


class I8FeedForward:
    """The feed-forward block with its products in 8-bit integers; b2c_hip_i8_ffn."""

    def __init__(self, x, w_gate, s_gate, w_up, s_up, w_down, s_down, y, act="silu", room=None):
        L = _lib()
        x = _floating(matrix(x, "x"), "x")
        g = matrix(w_gate, "w_gate", None, x.cols, I8)
        u = matrix(w_up, "w_up", g.rows, x.cols, I8)
        d = matrix(w_down, "w_down", None, g.rows, I8)
        if g.ld != u.ld:
            raise ValueError("i8_ffn: w_gate and w_up have different distances between rows")
        y = matrix(y, "y", x.rows, d.rows, x.dtype)
        a = self.args = I8FfnArgs(rows=x.rows, d_in=x.cols, d_hidden=g.rows, d_out=d.rows, dtype=x.dtype, act=_act(act),
                                  x=x.ptr, ldx=x.ld, w_gate=g.ptr, w_up=u.ptr, ld_in=g.ld,
                                  s_gate=_vector(s_gate, "s_gate", g.rows), s_up=_vector(s_up, "s_up", g.rows),
                                  w_down=d.ptr, ld_out=d.ld, s_down=_vector(s_down, "s_down", d.rows), y=y.ptr, ldy=y.ld)
        self._fn, self._ref = L.b2c_hip_i8_ffn, C.byref(a)
        a.workspace_bytes = L.b2c_i8_ffn_workspace_bytes(self._ref)
        b, a.workspace = _get_room(room, a.workspace_bytes, "i8_ffn")
        self._keep = (x, g, u, d, s_gate, s_up, s_down, y, b)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "i8_ffn")


def _weights(what, name, n, types):
    """The pointer and type of a norm's n weights, which lie next to each other."""
    if isinstance(what, Matrix):
        m, fits = what, what.rows * what.cols == n and (what.rows <= 1 or what.ld == what.cols)
    else:
        try:
            fits = tuple(what.shape) == (n,) and (n <= 1 or what.stride(0) == 1)
            if getattr(what, "is_cuda", True) is False:
                raise ValueError(f"{name}: is not on the GPU")
            m = Matrix(what.data_ptr(), n, 1, 1, NAMES.get(str(what.dtype).replace("torch.", "")), keep=what)
        except AttributeError:
            raise ValueError(f"{name}: {n} values are wanted, got {type(what).__name__}") from None
    if m.dtype not in types or not fits:
        raise ValueError(f"{name}: {n} values next to each other are wanted, of the matrices' type or in single precision")
    if not m.ptr:
        raise ValueError(f"{name}: a null pointer")
    return m


class BlockNorm:
    """Between two blocks: y = residual + scale act(gate) t with t = norm(x) w_post (`post`; else x itself), and n = norm(y) w_pre;
    b2c_hip_block_norm. What is not given is left out: without x, n is the norm of the residual, without a residual it counts as
    zeros, without n only y is formed. kind: rms or layer; gate_act: none or sigmoid. `gate` has a row for every `rows_per_gate` rows
    (by default: one row for all, or one for each). The weights are of the matrices' type or in single precision, both the same. y may be
    residual and n may be x, where no backward pass follows: that forms y again from x and residual."""

    def __init__(self, x=None, residual=None, y=None, n=None, gate=None, rows_per_gate=None, gate_act="none", post=False, w_post=None,
                 w_pre=None, kind="rms", eps=1e-6, scale=1.0):
        L = _lib()
        if x is None and residual is None:
            raise ValueError("block norm: needs x or residual")
        first = _floating(matrix(x if x is not None else residual, "x" if x is not None else "residual"), "x")
        m, d, t = first.rows, first.cols, first.dtype
        same = lambda what, name: matrix(what, name, m, d, t) if what is not None else None  # noqa: E731
        x, r, y, n = same(x, "x"), same(residual, "residual"), same(y, "y"), same(n, "n")
        if d > 16384:
            raise ValueError(f"block norm: {d} columns, at most 16384")
        if kind not in NORMS or gate_act not in GATES:
            raise ValueError(f"block norm: kind {kind!r} of {', '.join(NORMS)}, gate_act {gate_act!r} of {', '.join(GATES)}")
        if not 0.0 <= float(eps) < float("inf"):
            raise ValueError(f"block norm: eps {eps}")
        if x is None and (post or gate is not None or y is not None):
            raise ValueError("block norm: `post`, a gate and y need x")
        if w_post is not None and not post:
            raise ValueError("block norm: w_post without `post`")
        if w_pre is not None and n is None:
            raise ValueError("block norm: w_pre without n")
        if y is None and n is None:
            raise ValueError("block norm: neither y nor n is wanted")
        g = matrix(gate, "gate", None, d, t) if gate is not None else None
        if g is not None:
            if rows_per_gate is None:
                if g.rows not in (1, m):
                    raise ValueError("gate: rows_per_gate is needed")
                rows_per_gate = 1 if g.rows == m else max(m, 1)
            if rows_per_gate < 1 or g.rows < -(-m // rows_per_gate):
                raise ValueError(f"gate: has {g.rows} rows for {m} rows, {rows_per_gate} to each")
        elif rows_per_gate is not None:
            raise ValueError("block norm: rows_per_gate without a gate")
        ws = [_weights(w, name, d, (t, F32)) if w is not None else None for w, name in ((w_post, "w_post"), (w_pre, "w_pre"))]
        types = {w.dtype for w in ws if w}
        if len(types) > 1:
            raise ValueError("block norm: w_post and w_pre have different types")
        self._keep, self._shape, self._types = (x, r, g, ws, y, n), (m, d), (t, types.pop() if types else t)
        self._post, self._gate_rows = bool(post), -(-m // rows_per_gate) if g is not None else 0
        a = self.args = BlockNormArgs(rows=m, cols=d, dtype=t, w_dtype=self._types[1], kind=NORMS[kind], post=int(self._post),
                                      gate_act=GATES[gate_act], eps=eps, scale=scale, rows_per_gate=rows_per_gate or 0)
        for field, ld, v in (("x", "ldx", x), ("residual", "ldr", r), ("gate", "ldg", g), ("y", "ldy", y), ("n", "ldn", n)):
            setattr(a, field, v.ptr if v else None)
            setattr(a, ld, v.ld if v else 0)
        a.w_post, a.w_pre = (w.ptr if w else None for w in ws)
        self._ref, self._fwd, self._bwd = C.byref(a), L.b2c_hip_block_norm, L.b2c_hip_block_norm_backward
        self.grad = None

    def gradients(self, dy=None, dn=None, dx=None, dresidual=None, dgate=None, dw_post=None, dw_pre=None, accumulate=False, room=None):
        """Plans backward(): the gradients of y and n in (either may be missing), and whichever outputs are given. Those of the weights
        are of the weights' type, or in single precision, where `accumulate` adds to what they hold. dresidual may be dy and dx may be dn."""
        m, d = self._shape
        t, wt = self._types
        x, r, gate = self._keep[:3]
        if dy is None and dn is None:
            raise ValueError("block norm: needs dy or dn")
        if dn is None and dw_pre is not None:
            raise ValueError("block norm: dw_pre without dn")
        if x is None and dx is not None or gate is None and dgate is not None or not self._post and dw_post is not None:
            raise ValueError("block norm: a gradient of what was not given")
        same = lambda what, name: matrix(what, name, m, d, t) if what is not None else None  # noqa: E731
        dy, dn, dx, dr = same(dy, "dy"), same(dn, "dn"), same(dx, "dx"), same(dresidual, "dresidual")
        dg = matrix(dgate, "dgate", self._gate_rows, d, t) if dgate is not None else None
        ws = [_weights(w, name, d, (wt, F32)) if w is not None else None for w, name in ((dw_post, "dw_post"), (dw_pre, "dw_pre"))]
        types = {w.dtype for w in ws if w}
        if len(types) > 1:
            raise ValueError("block norm: dw_post and dw_pre have different types")
        kind = types.pop() if types else F32
        if accumulate and kind != F32:
            raise ValueError("block norm: gradients accumulate in single precision only")
        g = self.grad = BlockNormGradArgs(fwd=self.args, grad_dtype=kind, accumulate=int(bool(accumulate)))
        for field, ld, v in (("dy", "lddy", dy), ("dn", "lddn", dn), ("dx", "lddx", dx), ("dresidual", "lddr", dr), ("dgate", "lddg", dg)):
            setattr(g, field, v.ptr if v else None)
            setattr(g, ld, v.ld if v else 0)
        g.dw_post, g.dw_pre = (w.ptr if w else None for w in ws)
        self._gref = C.byref(g)
        g.workspace_bytes = _lib().b2c_block_norm_grad_workspace_bytes(self._gref)
        b, g.workspace = _get_room(room, g.workspace_bytes, "block norm gradients")
        self._gkeep = [dy, dn, dx, dr, dg, ws, b]

    def forward(self, stream=0):
        _check(self._fwd(self._ref, stream), "block norm")

    def backward(self, stream=0):
        if self.grad is None:
            raise ValueError("block norm: plan gradients() first")
        _check(self._bwd(self._gref, stream), "block norm gradients")


def _group(group):
    if group not in GROUPS:
        raise ValueError(f"group of {group} columns: wanted one of {', '.join(map(str, GROUPS))}")
    return group


def _near(*matrices):
    for m in matrices:
        if m is not None and m.ld > 1 << 25:
            raise ValueError(f"rows {m.ld} values apart: at most {1 << 25} for weights here")


class QuantizeGroups:
    """q, scale (and with `zero` zero points) = x in 4 bits, a scale for every `group` columns of a row; b2c_hip_quantize4. q is uint8,
    two columns a byte, the even one in the low half; `scale` is in 16 bits. `values`: what the codes stand for, of x's type. For weights
    [outputs, inputs], rows are channels."""

    def __init__(self, x, q, scale, group, zero=None, values=None):
        x = _floating(matrix(x, "x"), "x")
        n = -(-x.cols // _group(group))
        q = matrix(q, "q", x.rows, -(-x.cols // 2), U8)
        s = _floating(matrix(scale, "scale", x.rows, n), "scale", (F16, BF16))
        z = matrix(zero, "zero", x.rows, n, U8) if zero is not None else None
        v = matrix(values, "values", x.rows, x.cols, x.dtype) if values is not None else None
        self._keep = (x, q, s, z, v)
        self.args = Quantize4Args(rows=x.rows, cols=x.cols, group=group, dtype=x.dtype, scale_dtype=s.dtype, x=x.ptr, ldx=x.ld, q=q.ptr,
                                  ldq=q.ld, scale=s.ptr, lds=s.ld, zero=z.ptr if z else None, ldz=z.ld if z else 0,
                                  values=v.ptr if v else None, ldv=v.ld if v else 0)
        self._fn, self._ref = _lib().b2c_hip_quantize4, C.byref(self.args)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "quantize4")


class Q4Linear:
    """y = x w' with w held in 4 bits as QuantizeGroups gives it, its scales of x's type; b2c_hip_q4_linear."""

    def __init__(self, x, w, scale, y, group, zero=None, room=None):
        L = _lib()
        x = _floating(matrix(x, "x"), "x", (F16, BF16))
        n = -(-x.cols // _group(group))
        w = matrix(w, "w", None, -(-x.cols // 2), U8)
        s = matrix(scale, "scale", w.rows, n, x.dtype)
        z = matrix(zero, "zero", w.rows, n, U8) if zero is not None else None
        y = matrix(y, "y", x.rows, w.rows, x.dtype)
        _near(w, s, z)
        a = self.args = Q4LinearArgs(rows=x.rows, d_in=x.cols, d_out=w.rows, group=group, dtype=x.dtype, x=x.ptr, ldx=x.ld, w=w.ptr,
                                     ldw=w.ld, scale=s.ptr, lds=s.ld, zero=z.ptr if z else None, ldz=z.ld if z else 0, y=y.ptr, ldy=y.ld)
        self._fn, self._ref = L.b2c_hip_q4_linear, C.byref(a)
        a.workspace_bytes = L.b2c_q4_linear_workspace_bytes(self._ref)
        b, a.workspace = _get_room(room, a.workspace_bytes, "q4_linear")
        self._keep = (x, w, s, z, y, b)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "q4_linear")


class Experts:
    """A mixture of experts for a few tokens: y = residual + the sum over a row's `top_k` experts of p w_down (act(w_gate x) * (w_up x)), p the
    router's softmax, with `normalize` over the chosen ones alone; b2c_hip_experts. w_router is [experts, inputs]; w_gate and w_up hold one
    expert's [hidden, inputs] after the other's as rows, w_down their [outputs, hidden]. index (int32) and weight (single precision),
    [rows, top_k], take the choice, the largest first. y may be residual."""

    def __init__(self, x, w_router, w_gate, w_up, w_down, y, top_k, act="silu", normalize=True, residual=None, index=None, weight=None,
                 room=None):
        L = _lib()
        x = _floating(matrix(x, "x"), "x", (F16, BF16))
        t, m = x.dtype, x.rows
        wr = matrix(w_router, "w_router", None, x.cols, t)
        g, u = matrix(w_gate, "w_gate", None, x.cols, t), matrix(w_up, "w_up", None, x.cols, t)
        e = wr.rows
        if not 1 <= e <= 1024 or not 1 <= top_k <= min(e, 64):
            raise ValueError(f"experts: {top_k} of {e}; wanted 1 to 64 of at most 1024")
        if g.rows < 1 or g.rows % e or u.rows != g.rows:
            raise ValueError(f"experts: w_gate and w_up have {g.rows} and {u.rows} rows for {e} experts")
        if g.ld != u.ld:
            raise ValueError("experts: w_gate and w_up have different distances between rows")
        y = matrix(y, "y", m, None, t)
        d = matrix(w_down, "w_down", e * y.cols, g.rows // e, t)
        r = matrix(residual, "residual", m, y.cols, t) if residual is not None else None
        _near(g, d)
        i = matrix(index, "index", m, top_k, I32) if index is not None else None
        w = matrix(weight, "weight", m, top_k, F32) if weight is not None else None
        a = self.args = ExpertsArgs(rows=m, d_in=x.cols, d_hidden=g.rows // e, d_out=y.cols, experts=e, top_k=top_k, dtype=t, act=_act(act),
                                    normalize=int(bool(normalize)), x=x.ptr, ldx=x.ld, w_router=wr.ptr, ld_router=wr.ld, w_gate=g.ptr,
                                    w_up=u.ptr, ld_in=g.ld, w_down=d.ptr, ld_out=d.ld, residual=r.ptr if r else None,
                                    ldr=r.ld if r else 0, y=y.ptr, ldy=y.ld, index=i.ptr if i else None, ldi=i.ld if i else 0,
                                    weight=w.ptr if w else None, ldw=w.ld if w else 0)
        self._fn, self._ref = L.b2c_hip_experts, C.byref(a)
        a.workspace_bytes = L.b2c_experts_workspace_bytes(self._ref)
        b, a.workspace = _get_room(room, a.workspace_bytes, "experts")
        self._keep = (x, wr, g, u, d, y, r, i, w, b)

    def run(self, stream=0):
        _check(self._fn(self._ref, stream), "experts")
