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

_TORCH_CODE = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
_NUMPY_CODE = {"float32": 0, "float16": 1}


def _bad(msg):
    return ZjaiError(_lib.INVALID_ARGUMENT, msg)


def _is_torch(a):
    return type(a).__module__.startswith("torch")


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
    """The buffers of one call: their pointers, that they lie on one side, the stream order."""

    def __init__(self, engine):
        self.engine, self.mem, self.device = engine, None, None

    def _side(self, a, what, code):
        if _is_torch(a):
            if not a.is_cuda or a.device.index != self.engine.device:
                raise _bad("%s must be a CUDA tensor of the engine's GPU" % what)
            if not a.is_contiguous():
                raise _bad("%s must be contiguous" % what)
            ptr, mem = a.data_ptr(), _lib.MEM_DEVICE
            self.device = a.device
        elif isinstance(a, np.ndarray):
            if not a.flags.c_contiguous:
                raise _bad("%s must be contiguous" % what)
            ptr, mem = a.ctypes.data, _lib.MEM_HOST
        else:
            raise _bad("%s must be a numpy array or a CUDA tensor" % what)
        if code is None:
            raise _bad("%s has an element type that is not taken" % what)
        if self.mem is None:
            self.mem = mem
        elif self.mem != mem:
            raise _bad("mixed host and device arguments")
        return ptr

    def map(self, a, what, shape=None, code=None):
        """(pointer, dtype code) of a map, checked against a shape and a type if given."""
        if a is None:
            raise _bad("%s is missing" % what)
        dt = getattr(a, "dtype", None)
        got = (_TORCH_CODE if _is_torch(a) else _NUMPY_CODE).get(str(dt))
        ptr = self._side(a, what, got)
        if code is not None and got != code:
            raise _bad("%s has another element type" % what)
        if shape is not None and tuple(a.shape) != shape:
            raise _bad("%s has shape %s, expected %s" % (what, tuple(a.shape), shape))
        return ptr, got

    def param(self, a, what, c):
        return self.map(a, what, (c,), 0)[0]

    def tape(self, t, what, shape=None):
        """zjai_tape of a Tape, checked against a map's shape."""
        if not isinstance(t, Tape):
            raise _bad("%s must be a Tape" % what)
        for a in (t.codes, t.exps):
            if str(getattr(a, "dtype", None)).split(".")[-1] != "int8":
                raise _bad("a tape's codes and exps are int8")
        codes = self._side(t.codes, what + ".codes", 0)
        exps = self._side(t.exps, what + ".exps", 0)
        got = tuple(t.codes.shape)
        if len(got) not in (3, 4) or (shape is not None and got != shape):
            raise _bad("%s has shape %s, expected %s" % (what, got, shape or "[(n,) c, h, w]"))
        if tuple(t.exps.shape) != _exps_shape(got):
            raise _bad("%s: exps have shape %s, expected %s" % (what, tuple(t.exps.shape),
                                                               _exps_shape(got)))
        return _lib.TapeC(codes, exps)

    def empty(self, shape, like, dtype=None):
        if _is_torch(like):
            import torch
            return torch.empty(shape, dtype=dtype or like.dtype, device=like.device)
        return np.empty(shape, dtype or like.dtype)

    def new_tape(self, shape, like):
        i8 = np.int8
        if _is_torch(like):
            import torch
            i8 = torch.int8
        return Tape(self.empty(shape, like, i8), self.empty(_exps_shape(shape), like, i8))

    def floats(self, shape, like):
        if _is_torch(like):
            import torch
            return torch.empty(shape, dtype=torch.float32, device=like.device)
        return np.empty(shape, np.float32)

    def __call__(self, f, *args):
        """f(engine, *args, mem), in order with torch's current stream."""
        if self.mem == _lib.MEM_DEVICE:
            import torch
            cur = torch.cuda.current_stream(self.device).cuda_stream or STREAM_LEGACY
            if cur != self.engine.stream:
                L, h = _lib.lib(), self.engine.handle
                check(L.zjai_ctx_wait_stream(h, cur))
                check(f(h, *args, self.mem))
                check(L.zjai_ctx_release_stream(h, cur))
                return
        check(f(self.engine.handle, *args, self.mem))


def _exps_shape(shape):
    return tuple(shape[:-2]) + (-(-(shape[-2] * shape[-1]) // GROUP),)


def _dims(shape, what):
    if len(shape) not in (3, 4):
        raise _bad("%s must be [c, h, w] or [n, c, h, w]" % what)
    return tuple(shape) if len(shape) == 4 else (1,) + tuple(shape)


def tape_pack(engine, x):
    """`Engine.tape_pack`."""
    call = _Call(engine)
    px, dt = call.map(x, "x")
    n, c, h, w = _dims(tuple(x.shape), "x")
    t = call.new_tape(tuple(x.shape), x)
    call(_lib.lib().zjai_tape_pack, px, dt, n, c, h, w,
         ctypes.byref(_lib.TapeC(call._side(t.codes, "codes", 0), call._side(t.exps, "exps", 0))))
    return t


def tape_unpack(engine, tape, dtype=None):
    """`Engine.tape_unpack`."""
    call = _Call(engine)
    tc = call.tape(tape, "tape")
    if dtype is None:
        if _is_torch(tape.codes):
            import torch
            dtype = torch.float32
        else:
            dtype = np.float32
    x = call.empty(tape.shape, tape.codes, dtype)
    px, dt = call.map(x, "the unpacked map")
    n, c, h, w = _dims(tape.shape, "tape")
    call(_lib.lib().zjai_tape_unpack, ctypes.byref(tc), n, c, h, w, px, dt)
    return x


def _params(call, c, post, scale, pre):
    prm = _lib.ResidualParams()
    for name, pair in (("post", post), ("pre", pre)):
        if pair is not None:
            if not isinstance(pair, (tuple, list)) or len(pair) != 2:
                raise _bad("%s is a pair (weight, bias)" % name)
            setattr(prm, name + "_weight", call.param(pair[0], name + " weight", c))
            setattr(prm, name + "_bias", call.param(pair[1], name + " bias", c))
    if scale is not None:
        prm.scale = call.param(scale, "scale", c)
    return prm


def _gate_shape(gate, shape):
    """Shape of the gate's map: the branch's, or one channel."""
    got = tuple(gate.shape)
    one = shape[:-3] + (1,) + shape[-2:]
    if got != shape and got != one:
        raise _bad("gate has shape %s, expected %s or %s" % (got, shape, one))
    return got


def gated_residual_norm(engine, x, f, post=None, gate=None, scale=None, pre=None, tape=()):
    """`Engine.gated_residual_norm`."""
    call = _Call(engine)
    px, dt = call.map(x, "x")
    shape = tuple(x.shape)
    n, c, h, w = _dims(shape, "x")
    pf = call.map(f, "f", shape, dt)[0]
    pg, gc, gshape = None, 0, None
    if gate is not None:
        gshape = _gate_shape(gate, shape)
        pg, gc = call.map(gate, "gate", gshape, dt)[0], gshape[-3]
    prm = _params(call, c, post, scale, pre)
    y = call.empty(shape, x)
    z = call.empty(shape, x) if pre is not None else None
    tapes, tc = {}, _lib.ResidualTapes()
    for name in tape:
        if name not in ("f", "gate", "y", "z"):
            raise _bad("tape names are f, gate, y and z")
        if (name == "gate" and gate is None) or (name == "z" and pre is None):
            continue
        tapes[name] = t = call.new_tape(gshape if name == "gate" else shape, x)
        setattr(tc, name, call.tape(t, name))
    call(_lib.lib().zjai_gated_residual_norm, px, pf, pg, gc, dt, n, c, h, w, ctypes.byref(prm),
         call.map(y, "y")[0], call.map(z, "z")[0] if z is not None else None,
         ctypes.byref(tc) if tapes else None)
    return y, z, tapes


def gated_residual_norm_backward(engine, dy, dz=None, f=None, y=None, post=None, gate=None,
                                 scale=None, pre=None):
    """`Engine.gated_residual_norm_backward`."""
    call = _Call(engine)
    pdy, dt = call.map(dy, "dy")
    shape = tuple(dy.shape)
    n, c, h, w = _dims(shape, "dy")
    pdz = call.map(dz, "dz", shape, dt)[0] if pre is not None else None
    if dz is not None and pre is None:
        raise _bad("dz without pre")
    prm = _params(call, c, post, scale, pre)
    need_f = post is not None or scale is not None or gate is not None
    kept = {"f": f if need_f else None, "gate": gate, "y": y if pre is not None else None}
    for name, needed in (("f", need_f), ("y", pre is not None)):
        if needed and kept[name] is None:
            raise _bad("%s is missing" % name)
    used = [v for v in kept.values() if v is not None]
    taped = bool(used) and isinstance(used[0], Tape)
    if any(isinstance(v, Tape) != taped for v in used):
        raise _bad("f, gate and y are all Tapes or all maps")
    gshape = _gate_shape(gate, shape) if gate is not None else None
    ptr, tc = {}, _lib.ResidualTapes()
    for name, v in kept.items():
        ptr[name] = None
        if v is None:
            continue
        want = gshape if name == "gate" else shape
        if taped:
            setattr(tc, name, call.tape(v, name, want))
        else:
            ptr[name] = call.map(v, name, want, dt)[0]
    out = {"x": call.empty(shape, dy), "f": call.empty(shape, dy)}
    if gate is not None:
        out["gate"] = call.empty(gshape, dy)
    names = [k for k, on in (("post_weight", post), ("post_bias", post), ("scale", scale),
                             ("pre_weight", pre), ("pre_bias", pre)) if on is not None]
    for k in names:
        out[k] = call.floats((c,), dy)
    gr = _lib.ResidualGrads()
    for k, v in out.items():
        setattr(gr, k, call.map(v, k)[0])
    call(_lib.lib().zjai_gated_residual_norm_backward, pdy, pdz, ptr["f"], ptr["gate"],
         gshape[-3] if gshape else 0, ptr["y"], ctypes.byref(tc) if taped else None, dt, n, c, h, w,
         ctypes.byref(prm), ctypes.byref(gr))
    return out


def conv1x1_weight_grad(engine, dout, tape):
    """`Engine.conv1x1_weight_grad`."""
    call = _Call(engine)
    pd, dt = call.map(dout, "dout")
    n, oc, h, w = _dims(tuple(dout.shape), "dout")
    if not isinstance(tape, Tape):
        raise _bad("the input must be a Tape")
    c = tape.shape[-3] if len(tape.shape) in (3, 4) else 0
    tc = call.tape(tape, "tape", tuple(dout.shape[:-3]) + (c, h, w))
    dw, db = call.floats((oc, c), dout), call.floats((oc,), dout)
    call(_lib.lib().zjai_conv1x1_weight_grad, pd, dt, n, oc, c, h, w, ctypes.byref(tc),
         call.map(dw, "dw")[0], call.map(db, "db")[0])
    return dw, db
