"""8-bit activation tapes and the training operators that write and read them, as methods of
`Engine` (over `zjai_tape_*`, `zjai_gated_residual_norm*` and `zjai_conv1x1_weight_grad`).

Maps are `[c, h, w]` or `[n, c, h, w]`: numpy arrays (float32, float16) or CUDA tensors of the
engine's GPU (float32, float16, bfloat16), contiguous. Parameters are float32 of the same side.

CUDA tensors may be in use on torch's current stream, whichever that is: where the engine works on
another stream, its work is ordered after what the current stream holds and before what it is given
next. An engine set to the current stream (`set_stream`; `STREAM_LEGACY` is torch's default one)
spares a call that ordering.
"""

import ctypes

import numpy as np

from . import _lib
from ._lib import ZjaiError, check

GROUP = 32  # positions that share an exponent
STREAM_LEGACY = 1  # CUDA's handle of the legacy default stream, for `Engine.set_stream`

_NUMPY_CODE = {np.dtype(np.float32): 0, np.dtype(np.float16): 1}
_F32, _I8 = np.dtype(np.float32), np.dtype(np.int8)
_torch, _torch_code, _current_stream, _Tensor = None, {}, None, ()


def _bad(msg):
    return ZjaiError(_lib.INVALID_ARGUMENT, msg)


def _is_torch(a):
    """Whether a is a torch tensor; torch is imported when the first one comes."""
    global _torch, _torch_code, _current_stream, _Tensor
    if _torch is None:
        if isinstance(a, np.ndarray) or not type(a).__module__.startswith("torch"):
            return False
        import torch
        _torch, _Tensor = torch, torch.Tensor
        _torch_code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        # the handle of torch's current stream; the raw form makes no Stream object (3 us a call)
        _current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream)
    return isinstance(a, _Tensor)


class Tape:
    """A map held in 8 bits: `codes` (int8, the map's shape) and `exps` (int8, one per group of 32
    positions of a channel row: [.., c, ceil(h w / 32)]). A position's value is code 2^e; e = 127
    marks a group that held an infinity or a NaN. `Engine.tape_pack` makes one."""

    __slots__ = ("codes", "exps")

    def __init__(self, codes, exps):
        self.codes, self.exps = codes, exps

    @property
    def shape(self):
        return tuple(self.codes.shape)


class _Call:
    """The buffers of one call: the side they lie on (that of `like`), their checks, their pointers
    and new ones like them, and the stream order."""

    __slots__ = ("engine", "device", "cuda", "f32", "i8", "like", "shape", "groups")

    def __init__(self, engine, like):
        self.engine, self.like, self.shape, self.groups = engine, like, None, None
        self.cuda = isinstance(like, _Tensor) or _is_torch(like)
        if self.cuda:
            self.f32, self.i8, self.device = _torch.float32, _torch.int8, engine.device
            if like.get_device() != engine.device:
                raise _bad("torch tensors must be CUDA tensors of the engine's GPU")
        elif isinstance(like, np.ndarray):
            self.f32, self.i8 = _F32, _I8
        else:
            raise _bad("arguments are numpy arrays or CUDA tensors")

    def code(self, a, what):
        """Element type of a map."""
        code = (_torch_code if self.cuda else _NUMPY_CODE).get(a.dtype)
        if code is None:
            raise _bad("%s has an element type that is not taken" % what)
        return code

    def ptr(self, a, what, shape, dtype):
        """Pointer of an array that must have this shape and type and lie with the others."""
        if self.cuda:
            # most of a small call's time is spent here: what is wrong is looked at afterwards
            if (isinstance(a, _Tensor) and a.dtype is dtype and a.shape == shape
                    and a.is_contiguous() and a.get_device() == self.device):
                return a.data_ptr()
            if not isinstance(a, _Tensor) or a.get_device() != self.device:
                raise _bad("%s must be a tensor of the same GPU" % what)
            contiguous = a.is_contiguous()
        else:
            if not isinstance(a, np.ndarray):
                raise _bad("%s must be a numpy array like the others" % what)
            contiguous = a.flags.c_contiguous
        if a.dtype != dtype:
            raise _bad("%s has type %s, expected %s" % (what, a.dtype, dtype))
        if tuple(a.shape) != tuple(shape):
            raise _bad("%s has shape %s, expected %s" % (what, tuple(a.shape), tuple(shape)))
        if not contiguous:
            raise _bad("%s must be contiguous" % what)
        return a.data_ptr() if self.cuda else a.ctypes.data

    def param(self, a, what, c):
        return self.ptr(a, what, (c,), self.f32)

    def tape(self, t, what, shape):
        """zjai_tape of a Tape of a map of this shape."""
        if not isinstance(t, Tape):
            raise _bad("%s must be a Tape" % what)
        return _lib.TapeC(self.ptr(t.codes, what, shape, self.i8),
                          self.ptr(t.exps, what, self.exps_shape(shape), self.i8))

    def exps_shape(self, shape):
        if shape == self.shape:
            return self.groups
        groups = -(-(shape[-2] * shape[-1]) // GROUP)
        self.shape, self.groups = shape, tuple(shape[:-2]) + (groups,)
        return self.groups

    def empty(self, shape, dtype):
        if self.cuda:
            return self.like.new_empty(shape, dtype=dtype)
        return np.empty(shape, dtype)

    def empty_like(self, dtype=None):
        """A map like the one that the call began with (of an element type)."""
        empty = _torch.empty_like if self.cuda else np.empty_like
        return empty(self.like, dtype=dtype)

    def at(self, a):
        """Pointer of an array of `empty`."""
        return a.data_ptr() if self.cuda else a.ctypes.data

    def new_tape(self, shape, like=False):
        """A tape of a map of this shape (like: that of the map that the call began with)."""
        codes = self.empty_like(self.i8) if like else self.empty(shape, self.i8)
        t = Tape(codes, self.empty(self.exps_shape(shape), self.i8))
        return t, _lib.TapeC(self.at(t.codes), self.at(t.exps))

    def __call__(self, f, *args):
        """f(engine, *args, mem), in order with torch's current stream."""
        if not self.cuda:
            check(f(self.engine.handle, *args, _lib.MEM_HOST))
            return
        h = self.engine.handle
        cur = _current_stream(self.engine.device) or STREAM_LEGACY
        if cur == self.engine.stream:
            check(f(h, *args, _lib.MEM_DEVICE))
            return
        L = _lib.lib()
        check(L.zjai_ctx_wait_stream(h, cur))
        check(f(h, *args, _lib.MEM_DEVICE))
        check(L.zjai_ctx_release_stream(h, cur))


def _dims(shape, what):
    """(n, c, h, w) of a map's shape."""
    if len(shape) == 4:
        return shape
    if len(shape) != 3:
        raise _bad("%s must be [c, h, w] or [n, c, h, w]" % what)
    return (1,) + tuple(shape)


def tape_pack(engine, x):
    """`Engine.tape_pack`."""
    call = _Call(engine, x)
    shape = x.shape
    n, c, h, w = _dims(shape, "x")
    px = call.ptr(x, "x", shape, x.dtype)
    code = call.code(x, "x")
    t, tc = call.new_tape(tuple(shape), True)
    call(_lib.lib().zjai_tape_pack, px, code, n, c, h, w, ctypes.byref(tc))
    return t


def tape_unpack(engine, tape, dtype=None):
    """`Engine.tape_unpack`."""
    if not isinstance(tape, Tape):
        raise _bad("not a Tape")
    call = _Call(engine, tape.codes)
    shape = tape.shape
    n, c, h, w = _dims(shape, "tape")
    tc = call.tape(tape, "tape", shape)
    x = call.empty_like(dtype or call.f32)  # (the codes' shape)
    call(_lib.lib().zjai_tape_unpack, ctypes.byref(tc), n, c, h, w, call.at(x),
         call.code(x, "the unpacked map"))
    return x


def _params(call, c, post, scale, pre):
    prm = _lib.ResidualParams()
    if post is not None:
        weight, bias = _pair(post, "post")
        prm.post_weight = call.param(weight, "post weight", c)
        prm.post_bias = call.param(bias, "post bias", c)
    if scale is not None:
        prm.scale = call.param(scale, "scale", c)
    if pre is not None:
        weight, bias = _pair(pre, "pre")
        prm.pre_weight = call.param(weight, "pre weight", c)
        prm.pre_bias = call.param(bias, "pre bias", c)
    return prm


def _pair(p, what):
    if not isinstance(p, (tuple, list)) or len(p) != 2:
        raise _bad("%s is a pair (weight, bias)" % what)
    return p


def _gate_shape(gate, shape):
    """Shape of the gate's map: the branch's, or one channel."""
    got = tuple(gate.shape)
    if got != shape and got != shape[:-3] + (1,) + shape[-2:]:
        raise _bad("gate has shape %s, expected %s or one channel of it" % (got, shape))
    return got


def gated_residual_norm(engine, x, f, post=None, gate=None, scale=None, pre=None, tape=()):
    """`Engine.gated_residual_norm`."""
    call = _Call(engine, x)
    shape, dt = tuple(x.shape), x.dtype
    n, c, h, w = _dims(shape, "x")
    code = call.code(x, "x")
    px, pf = call.ptr(x, "x", shape, dt), call.ptr(f, "f", shape, dt)
    pg, gc = None, 0
    if gate is not None:
        gshape = _gate_shape(gate, shape)
        pg, gc = call.ptr(gate, "gate", gshape, dt), gshape[-3]
    prm = _params(call, c, post, scale, pre)
    y = call.empty_like()
    z = call.empty_like() if pre is not None else None
    tapes, tc = {}, None
    for name in tape:
        if name not in ("f", "gate", "y", "z"):
            raise _bad("tape names are f, gate, y and z")
        if (name == "gate" and gate is None) or (name == "z" and pre is None):
            continue
        tc = tc or _lib.ResidualTapes()
        gates = name == "gate"
        tapes[name], one = call.new_tape(gshape if gates else shape, not gates or gshape == shape)
        setattr(tc, name, one)
    call(_lib.lib().zjai_gated_residual_norm, px, pf, pg, gc, code, n, c, h, w, ctypes.byref(prm),
         call.at(y), call.at(z) if z is not None else None, ctypes.byref(tc) if tc else None)
    return y, z, tapes


def gated_residual_norm_backward(engine, dy, dz=None, f=None, y=None, post=None, gate=None,
                                 scale=None, pre=None):
    """`Engine.gated_residual_norm_backward`."""
    call = _Call(engine, dy)
    shape, dt = tuple(dy.shape), dy.dtype
    n, c, h, w = _dims(shape, "dy")
    code = call.code(dy, "dy")
    pdy = call.ptr(dy, "dy", shape, dt)
    if (dz is None) != (pre is None):
        raise _bad("dz goes with pre")
    pdz = call.ptr(dz, "dz", shape, dt) if pre is not None else None
    prm = _params(call, c, post, scale, pre)
    gated = gate is not None
    need_f = gated or post is not None or scale is not None
    need_y = pre is not None
    gshape = _gate_shape(gate, shape) if gated else None
    taped = ((need_f and isinstance(f, Tape)) or (need_y and isinstance(y, Tape))
             or (gated and isinstance(gate, Tape)))
    for name, v, on in (("f", f, need_f), ("y", y, need_y)):
        if on and v is None:
            raise _bad("%s is missing" % name)
    pf = pg = py = tc = None
    if taped:  # all of them
        none = _lib.TapeC()
        tc = _lib.ResidualTapes(call.tape(f, "f", shape) if need_f else none,
                                call.tape(gate, "gate", gshape) if gated else none,
                                call.tape(y, "y", shape) if need_y else none)
    else:
        pf = call.ptr(f, "f", shape, dt) if need_f else None
        pg = call.ptr(gate, "gate", gshape, dt) if gated else None
        py = call.ptr(y, "y", shape, dt) if need_y else None
    dx, df = call.empty_like(), call.empty_like()
    out, pgate = {"x": dx, "f": df}, None
    if gated:
        out["gate"] = call.empty_like() if gshape == shape else call.empty(gshape, dt)
        pgate = call.at(out["gate"])
    rows, at = None, [None] * 5
    count = 2 * (post is not None) + (scale is not None) + 2 * need_y
    if count:  # rows of one array
        rows = call.empty((count, c), call.f32)
        first, rows = call.at(rows), iter(rows.unbind() if call.cuda else rows)
        for i, (name, on) in enumerate((("post_weight", post), ("post_bias", post), ("scale", scale),
                                        ("pre_weight", pre), ("pre_bias", pre))):
            if on is not None:
                out[name], at[i], first = next(rows), first, first + 4 * c
    gr = _lib.ResidualGrads(call.at(dx), call.at(df), pgate, *at)
    call(_lib.lib().zjai_gated_residual_norm_backward, pdy, pdz, pf, pg,
         gshape[-3] if gated else 0, py, ctypes.byref(tc) if taped else None, code, n, c, h,
         w, ctypes.byref(prm), ctypes.byref(gr))
    return out


def conv1x1_weight_grad(engine, dout, tape):
    """`Engine.conv1x1_weight_grad`."""
    call = _Call(engine, dout)
    shape = tuple(dout.shape)
    n, oc, h, w = _dims(shape, "dout")
    code = call.code(dout, "dout")
    pd = call.ptr(dout, "dout", shape, dout.dtype)
    if not isinstance(tape, Tape) or len(tape.shape) != len(shape):
        raise _bad("the input must be a Tape with dout's dimensions")
    c = tape.shape[-3]
    tc = call.tape(tape, "tape", shape[:-3] + (c, h, w))
    dw, db = call.empty((oc, c), call.f32), call.empty((oc,), call.f32)
    call(_lib.lib().zjai_conv1x1_weight_grad, pd, code, n, oc, c, h, w, ctypes.byref(tc),
         call.at(dw), call.at(db))
    return dw, db
