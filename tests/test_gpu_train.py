"""The training operators on the GPU through the public entry points against their definitions in 64
bits (train_reference.py): 8-bit tapes, the gated residual norm and its backward pass, the weight
gradient of a 1x1 convolution from a tape.

Tolerances, by derivation. Tapes are exact: equal. A map in f32 carries a dozen roundings of its own
2^-24 and a sum over the channels: 4e-6 relative L2; a map in f16 / bf16 is rounded once more at the
end: half a unit in the last place (2^-11, 2^-8) on top. Gradients are held per element to 4e-6 of
the formula's value with the magnitudes of all that it adds and subtracts (a few dozen roundings of
2^-24 each, and f32 sums), since norms and their gradients are differences that may cancel."""

import ctypes

import numpy as np
import pytest

import train_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
END = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
MAP_TOL = 4e-6
SUM_TOL = 4e-6


@pytest.fixture(scope="module")
def eng():
    import zenjpegai_b200 as zj
    e = zj.Engine(0, arena_bytes=1 << 28)
    yield e
    e.close()


def dev(a, dtype="f32"):
    return torch.from_numpy(np.asarray(a, np.float32)).cuda().to(DT[dtype])


def f64(t):
    return t.double().cpu().numpy()


def close(got, want, dtype, extra=0.0):
    g = f64(got)
    assert g.shape == want.shape
    err, norm = np.linalg.norm((g - want).ravel()), np.linalg.norm(want.ravel())
    # half a unit of f16's subnormals is absolute
    small = 2.0 ** -25 * np.sqrt(want.size) if dtype == "f16" else 0.0
    assert err <= (MAP_TOL + END[dtype] + extra) * norm + small, (err, norm)


def shifted(t):
    """The same contiguous map, one element off its allocation's alignment."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    v = buf[1:].view(t.shape)
    v.copy_(t)
    return v


def the_tape(codes, exps):
    import zenjpegai_b200 as zj
    return zj.Tape(torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda())


# ---- tapes -----------------------------------------------------------------------------------

SHAPES = [(1, 1, 1, 1), (1, 3, 1, 31), (2, 5, 4, 8), (1, 7, 3, 11), (3, 64, 33, 29), (2, 130, 16, 16),
          (1, 16, 1, 4097), (1, 2, 128, 128), (5, 3, 7, 160)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("off", [False, True])
def test_tape_round_trip(eng, shape, dtype, off):
    rng = np.random.default_rng(sum(shape))
    lo, hi = (-10, 5) if dtype == "f16" else (-60, 60)
    x = rng.standard_normal(shape) * np.exp2(rng.integers(lo, hi, shape))
    x[0, 0] *= 0.0
    t = dev(x, dtype)
    t = shifted(t) if off else t
    codes, exps = ref.pack(f64(t))
    tape = eng.tape_pack(t)
    assert np.array_equal(tape.codes.cpu().numpy(), codes)
    assert np.array_equal(tape.exps.cpu().numpy(), exps)
    want = ref.unpack(codes, exps)
    if off:
        tape.codes = shifted(tape.codes)
    for name in DT:
        got = eng.tape_unpack(tape, DT[name])
        if name == "f16":
            with np.errstate(over="ignore"):
                assert np.array_equal(f64(got), want.astype(np.float16).astype(np.float64))
        else:
            assert np.array_equal(f64(got), want)


def test_tape_edges(eng):
    x = np.zeros((1, 12, 1, 70), np.float32)
    x[0, 0, 0, 3] = np.inf
    x[0, 1, 0, 40] = -np.inf
    x[0, 2, 0, 69] = np.nan
    x[0, 3, 0, :] = 3.4e38                     # the largest
    x[0, 4, 0, :] = 1e-38                      # below 2^-120: the exponent's lower end
    x[0, 5, 0, :] = 1e-45
    x[0, 6, 0, :] = np.linspace(-128, 128, 70)  # ties and saturation at a step of 1 and 2
    x[0, 7, 0, :32] = np.arange(32) - 15.5
    x[0, 7, 0, 0] = 64
    x[0, 8, 0, :] = np.nextafter(np.float32(1), np.float32(0))
    x[0, 9, 0, :] = -1.0
    x[0, 10, 0, :] = 127.5
    x[0, 11, 0, 64:] = 65504.0
    codes, exps = ref.pack(x)
    tape = eng.tape_pack(dev(x))
    assert np.array_equal(tape.codes.cpu().numpy(), codes)
    assert np.array_equal(tape.exps.cpu().numpy(), exps)
    for name in ("f32", "bf16"):
        np.testing.assert_array_equal(f64(eng.tape_unpack(tape, DT[name])), ref.unpack(codes, exps))
    half = eng.tape_unpack(eng.tape_pack(dev(np.clip(x, -65504, 65504), "f16")), DT["f16"])
    assert not torch.isinf(half).any()  # the largest f16 does not round up to infinity


def test_host_arrays(eng):
    rng = np.random.default_rng(0)
    for dt in (np.float32, np.float16):
        x = rng.standard_normal((6, 9, 7)).astype(dt)
        t = eng.tape_pack(x)
        codes, exps = ref.pack(x[None])
        assert np.array_equal(t.codes, codes[0]) and np.array_equal(t.exps, exps[0])
        assert np.array_equal(eng.tape_unpack(t).astype(np.float64), ref.unpack(codes, exps)[0])
        w = (np.ones(6, np.float32), np.zeros(6, np.float32))
        y, z, tapes = eng.gated_residual_norm(x, x, pre=w, tape=("z",))
        wy, wz = ref.residual(x[None].astype(np.float64), x[None].astype(np.float64), pre=w)
        end = 2.0 ** -11 if dt == np.float16 else 0.0
        for g, want in ((y, wy[0]), (z, wz[0])):
            assert np.linalg.norm(g.astype(np.float64) - want) <= (4e-6 + end) * np.linalg.norm(want)
        g = eng.gated_residual_norm_backward(x, x, y=x, pre=w)
        assert g["x"].dtype == dt and g["pre_weight"].dtype == np.float32
        dw, db = eng.conv1x1_weight_grad(x, t)
        ww, wb = ref.weight_grad(x[None].astype(np.float64), ref.unpack(codes, exps))
        assert np.allclose(dw, ww, rtol=1e-4, atol=1e-4) and np.allclose(db, wb, rtol=1e-5, atol=1e-5)


# ---- gated residual norm ---------------------------------------------------------------------

def step_case(rng, shape, gate_channels, parts):
    n, c, h, w = shape
    spread = np.exp(0.7 * rng.standard_normal((1, c, 1, 1)))
    v = {"x": rng.standard_normal(shape) * spread + 0.3, "f": rng.standard_normal(shape) * spread - 1}
    kw = {"gate": rng.standard_normal((n, gate_channels, h, w)) * 3 if gate_channels else None,
          "scale": 0.5 + 0.1 * rng.standard_normal(c) if "s" in parts else None}
    for k, on in (("post", "p"), ("pre", "n")):
        kw[k] = ((1 + 0.2 * rng.standard_normal(c), 0.2 * rng.standard_normal(c))
                 if on in parts else None)
    return v, kw


def on_device(kw, dtype):
    return {"gate": dev(kw["gate"], dtype) if kw["gate"] is not None else None,
            "scale": dev(kw["scale"]) if kw["scale"] is not None else None,
            "post": tuple(map(dev, kw["post"])) if kw["post"] else None,
            "pre": tuple(map(dev, kw["pre"])) if kw["pre"] else None}


def as_f64(kw):
    one = lambda v: tuple(f64(a) for a in v) if isinstance(v, tuple) else f64(v)  # noqa: E731
    return {k: one(v) if v is not None else None for k, v in kw.items()}


STEPS = [((1, 128, 1, 1), "full", "psn"), ((2, 64, 16, 16), "full", "psn"),
         ((1, 160, 7, 13), "one", "psn"), ((3, 33, 5, 9), "full", "n"), ((1, 96, 3, 50), "none", "p"),
         ((2, 1, 4, 11), "one", "psn"), ((1, 2, 6, 6), "full", "ps"), ((1, 200, 9, 31), "one", "s"),
         ((1, 257, 5, 7), "full", "psn"), ((1, 515, 2, 33), "one", "pn"), ((1, 64, 8, 8), "none", ""),
         ((1, 1100, 1, 40), "full", "psn"), ((1, 2100, 1, 5), "none", "psn"), ((1, 16, 67, 61), "none", "sn")]


def gate_channels(kind, c):
    return {"full": c, "one": 1, "none": 0}[kind]


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype", list(DT))
def test_residual_norm(eng, shape, gate, parts, dtype):
    rng = np.random.default_rng(sum(shape) + len(parts))
    v, kw = step_case(rng, shape, gate_channels(gate, shape[1]), parts)
    x, f, dk = dev(v["x"], dtype), dev(v["f"], dtype), on_device(kw, dtype)
    y, z, tapes = eng.gated_residual_norm(x, f, tape=("f", "gate", "y", "z"), **dk)
    wy, wz = ref.residual(f64(x), f64(f), **as_f64(dk))
    close(y, wy, dtype)
    assert (z is None) == (wz is None)
    if z is not None:
        close(z, wz, dtype)
    assert set(tapes) == {"f", "y"} | ({"gate"} if gate != "none" else set()) | (
        {"z"} if z is not None else set())
    for name, src in (("f", f), ("gate", dk["gate"])):
        if name in tapes:
            codes, exps = ref.pack(f64(src))
            assert np.array_equal(tapes[name].codes.cpu().numpy(), codes)
            assert np.array_equal(tapes[name].exps.cpu().numpy(), exps)
    # y and z are rounded from values that differ from the definition's in the last places: a code
    # may be one off where the definition lies next to a tie, a value never more than a step
    for name, want in (("y", wy), ("z", wz)):
        if name not in tapes:
            continue
        codes, exps = ref.pack(want)
        got = ref.unpack(tapes[name].codes.cpu().numpy(), tapes[name].exps.cpu().numpy())
        step = np.repeat(np.exp2(exps.astype(np.float64)), 32, 2)[:, :, :shape[2] * shape[3]]
        assert (np.abs(got - want) <= 1.01 * step.reshape(want.shape)).all()
        assert np.mean(got != ref.unpack(codes, exps)) < 0.01
    again = eng.gated_residual_norm(shifted(x), shifted(f), **dk)
    assert torch.equal(again[0], y) and (z is None or torch.equal(again[1], z))


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("taped", [True, False])
def test_residual_norm_backward(eng, shape, gate, parts, dtype, taped):
    rng = np.random.default_rng(sum(shape) + len(parts))
    v, kw = step_case(rng, shape, gate_channels(gate, shape[1]), parts)
    dk = on_device(kw, dtype)
    f, y = dev(v["f"], dtype), dev(v["x"], dtype)
    dy = dev(rng.standard_normal(shape) * 1e-2, dtype)
    dz = dev(rng.standard_normal(shape) * 1e-2, dtype) if "n" in parts else None
    rk, kept = as_f64(dk), {"f": f, "y": y, "gate": dk["gate"]}
    rf, ry = f64(f), f64(y)
    if taped:
        held = {k: ref.pack(f64(a)) for k, a in kept.items() if a is not None}
        rf, ry = ref.unpack(*held["f"]), ref.unpack(*held["y"])
        if dk["gate"] is not None:
            rk["gate"] = ref.unpack(*held["gate"])
        kept = {k: the_tape(*held[k]) if k in held else None for k in kept}
    dk["gate"] = kept["gate"]
    want, mag = ref.residual_backward(f64(dy), f64(dz) if dz is not None else None, rf, ry, **rk)
    got = eng.gated_residual_norm_backward(dy, dz, f=kept["f"], y=kept["y"], **dk)
    assert set(got) == set(want)
    for k in got:
        end = END[dtype] if k in ("x", "f", "gate") else 0.0
        small = 2.0 ** -25 if end and dtype == "f16" else 0.0  # half a unit of f16's subnormals
        err = np.abs(f64(got[k]) - want[k])
        assert (err <= SUM_TOL * mag[k] + end * np.abs(want[k]) + small).all(), k
    again = eng.gated_residual_norm_backward(dy, dz, f=kept["f"], y=kept["y"], **dk)
    assert all(torch.equal(again[k], got[k]) for k in got)


def test_residual_norm_edges(eng):
    """Gate logits at the ends, a branch that is the same in all channels, a marked tape group."""
    c, shape = 8, (1, 8, 1, 40)
    x, f = np.zeros(shape), np.full(shape, 0.5)
    gate = np.zeros(shape)
    gate[0, :, 0, :6] = [np.inf, -np.inf, 90.0, -90.0, 200.0, -200.0]
    one = (np.ones(c), np.full(c, 2.0))
    y, z, _ = eng.gated_residual_norm(dev(x), dev(f), post=tuple(map(dev, one)), gate=dev(gate),
                                      pre=tuple(map(dev, one)))
    wy, wz = ref.residual(x, f, one, gate, None, one)
    assert np.allclose(f64(y), wy, rtol=1e-6, atol=1e-37) and np.allclose(f64(z), wz, rtol=1e-6)
    g = eng.gated_residual_norm_backward(dev(x + 1), dev(x), f=dev(f), y=dev(x), gate=dev(gate),
                                         post=tuple(map(dev, one)), pre=tuple(map(dev, one)))
    assert all(torch.isfinite(t).all() for t in g.values())
    sg = ref.sigmoid(gate)
    assert np.allclose(f64(g["gate"]), 2 * sg * (1 - sg), rtol=1e-6, atol=1e-12)
    # a NaN in one position stays in its position; on a tape in its group
    f[0, 3, 0, 35] = np.nan
    y, z, tapes = eng.gated_residual_norm(dev(x), dev(f), pre=tuple(map(dev, one)), tape=("f", "y"))
    bad = torch.isnan(z).any(1).view(-1).cpu().numpy()
    assert bad[35] and bad.sum() == 1
    assert tapes["f"].exps[0, 3].tolist() == [-7, 127]
    g = eng.gated_residual_norm_backward(dev(x), dev(x), f=tapes["f"], y=tapes["y"],
                                         scale=dev(np.ones(c)), pre=tuple(map(dev, one)))
    assert torch.isnan(g["x"]).any(1).view(-1).tolist() == [False] * 32 + [True] * 8


# ---- weight gradient ---------------------------------------------------------------------------

@pytest.mark.parametrize("n,oc,c,h,w", [(1, 1, 1, 1, 1), (1, 128, 128, 16, 16), (2, 200, 72, 11, 13),
                                        (1, 384, 128, 30, 64), (3, 16, 8, 5, 7), (1, 129, 257, 8, 48),
                                        (1, 96, 64, 1, 5000), (28, 64, 16, 4, 8), (2, 300, 40, 33, 29),
                                        (1, 128, 512, 64, 64)])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("off", [False, True])
def test_weight_grad(eng, n, oc, c, h, w, dtype, off):
    rng = np.random.default_rng(oc + c + h)
    codes, exps = ref.pack(rng.standard_normal((n, c, h, w)) * np.exp(rng.standard_normal((1, c, 1, 1))))
    d = dev(rng.standard_normal((n, oc, h, w)) * 1e-2, dtype)
    tape = the_tape(codes, exps)
    if off:
        d, tape.codes = shifted(d), shifted(tape.codes)
    dw, db = eng.conv1x1_weight_grad(d, tape)
    x = ref.unpack(codes, exps)
    ww, wb = ref.weight_grad(f64(d), x)
    mw, mb = ref.weight_grad(np.abs(f64(d)), np.abs(x))
    assert dw.dtype == db.dtype == torch.float32
    assert (np.abs(f64(dw) - ww) <= SUM_TOL * mw).all()
    assert (np.abs(f64(db) - wb) <= SUM_TOL * mb).all()
    again = eng.conv1x1_weight_grad(d, tape)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_weight_grad_edges(eng):
    """A marked group spoils its input channel alone, an infinity or NaN in d_out its output
    channel alone; tiny and huge gradients keep their precision."""
    rng = np.random.default_rng(5)
    codes, exps = ref.pack(rng.standard_normal((1, 40, 9, 11)) + 2)
    exps[0, 7, 1] = 127
    d = rng.standard_normal((1, 50, 9, 11)).astype(np.float32)
    d[0, 3, 4, 4] = np.inf
    d[0, 9, 0, 0] = np.nan
    dw, db = eng.conv1x1_weight_grad(dev(d), the_tape(codes, exps))
    dw, db = f64(dw), f64(db)
    spoiled = np.zeros((50, 40), bool)
    spoiled[9], spoiled[:, 7] = True, True
    assert np.isnan(dw[spoiled]).all() and np.isinf(np.delete(dw[3], 7)).all()
    spoiled[3] = True
    assert np.isfinite(dw[~spoiled]).all()
    assert np.isinf(db[3]) and np.isnan(db[9]) and np.isfinite(np.delete(db, [3, 9])).all()
    exps[0, 7, 1] = 0
    for mag in (1e-30, 1e30):
        d = rng.standard_normal((1, 50, 9, 11)) * mag
        dw, _ = eng.conv1x1_weight_grad(dev(d), the_tape(codes, exps))
        d = f64(dev(d))
        ww, _ = ref.weight_grad(d, ref.unpack(codes, exps))
        mw, _ = ref.weight_grad(np.abs(d), np.abs(ref.unpack(codes, exps)))
        assert (np.abs(f64(dw) - ww) <= SUM_TOL * mw).all()


# ---- streams, refusals -------------------------------------------------------------------------

def test_other_streams(eng):
    """Inputs written and outputs read on a torch stream while the engine works on its own."""
    rng = np.random.default_rng(6)
    host = torch.from_numpy(rng.standard_normal((4, 64, 96, 96)).astype(np.float32)).pin_memory()
    codes, exps = ref.pack(2 * host.numpy().astype(np.float64))
    for stream in (torch.cuda.Stream(), torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            for _ in range(8):
                x = host.cuda(non_blocking=True)
                x = x + x  # freed and reused by the next turn
                tape = eng.tape_pack(x)
                x.zero_()
                y = eng.tape_unpack(tape, torch.float32)
                got = y.clone()
                y.zero_()
        stream.synchronize()
        assert np.array_equal(f64(got), ref.unpack(codes, exps))
    # set to the caller's stream
    import zenjpegai_b200 as zj
    eng.set_stream(zj.STREAM_LEGACY)
    try:
        x = host.cuda()
        assert np.array_equal(f64(eng.tape_unpack(eng.tape_pack(x + x))), ref.unpack(codes, exps))
    finally:
        torch.cuda.synchronize()
        eng.set_stream(None)


def test_refusals(eng):
    from zenjpegai_b200 import _lib
    L, h = _lib.lib(), eng.handle
    x = torch.zeros(1, 4, 8, 8, device="cuda")
    t = eng.tape_pack(x)
    torch.cuda.synchronize()
    tc = _lib.TapeC(t.codes.data_ptr(), t.exps.data_ptr())
    host = np.zeros((1, 4, 8, 8), np.float32)
    D = _lib.MEM_DEVICE
    bad, big, un = _lib.INVALID_ARGUMENT, _lib.LIMIT_EXCEEDED, _lib.UNSUPPORTED
    px, tp = x.data_ptr(), ctypes.byref(tc)
    prm, gr = _lib.ResidualParams(), _lib.ResidualGrads()
    pp, pg = ctypes.byref(prm), ctypes.byref(gr)
    assert L.zjai_tape_pack(None, px, 0, 1, 4, 8, 8, tp, D) == bad
    assert L.zjai_tape_pack(h, px, 3, 1, 4, 8, 8, tp, D) == bad
    assert L.zjai_tape_pack(h, px, 0, 1, 4, 0, 8, tp, D) == bad
    assert L.zjai_tape_pack(h, px, 0, 1, 4, 8, 8, tp, 7) == bad
    assert L.zjai_tape_pack(h, None, 0, 1, 4, 8, 8, tp, D) == bad
    assert L.zjai_tape_pack(h, px, 0, 1, 4, 8, 8, None, D) == bad
    assert L.zjai_tape_pack(h, px + 2, 0, 1, 4, 8, 8, tp, D) == bad  # misaligned
    assert L.zjai_tape_pack(h, host.ctypes.data, 0, 1, 4, 8, 8, tp, D) == bad
    assert L.zjai_tape_pack(h, px, 0, 1, 4, 1 << 16, 1 << 16, tp, D) == big
    assert L.zjai_tape_pack(h, px, 0, 1 << 20, 1 << 20, 8, 8, tp, D) == big
    assert L.zjai_tape_unpack(h, tp, 1, 4, 8, 8, px + 1, 1, D) == bad
    assert L.zjai_gated_residual_norm(h, px, px, None, 0, 0, 1, 9000, 8, 8, pp, px, None, None, D) == un
    assert L.zjai_gated_residual_norm(h, px, px, px, 2, 0, 1, 4, 8, 8, pp, px, None, None, D) == bad
    assert L.zjai_gated_residual_norm(h, px, px, None, 4, 0, 1, 4, 8, 8, pp, px, None, None, D) == bad
    assert L.zjai_gated_residual_norm(h, px, px, None, 0, 0, 1, 4, 8, 8, None, px, None, None, D) == bad
    prm.pre_weight = px
    assert L.zjai_gated_residual_norm(h, px, px, None, 0, 0, 1, 4, 8, 8, pp, px, px, None, D) == bad
    prm.pre_bias = px
    assert L.zjai_gated_residual_norm(h, px, px, None, 0, 0, 1, 4, 8, 8, pp, px, None, None, D) == bad
    gr.x = gr.f = gr.pre_weight = px
    args = (0, 1, 4, 8, 8, pp, pg, D)
    assert L.zjai_gated_residual_norm_backward(h, px, px, None, None, 0, px, None, *args) == bad
    gr.pre_bias = px
    assert L.zjai_gated_residual_norm_backward(h, px, None, None, None, 0, px, None, *args) == bad
    assert L.zjai_gated_residual_norm_backward(h, px, px, None, None, 0, None, None, *args) == bad
    both = _lib.ResidualTapes()
    both.y = tc
    assert L.zjai_gated_residual_norm_backward(h, px, px, None, None, 0, px, ctypes.byref(both),
                                               *args) == bad
    assert L.zjai_conv1x1_weight_grad(h, px, 0, 1, 4, 4, 8, 8, tp, None, None, D) == bad
    assert L.zjai_conv1x1_weight_grad(h, px, 0, 1, 4, 4, 8, 8, None, px, None, D) == bad
    assert L.zjai_conv1x1_weight_grad(h, px, 0, 1, 0, 4, 8, 8, tp, px, None, D) == bad
    # a dw alone is a call
    dw = torch.empty(4, 4, device="cuda")
    torch.cuda.synchronize()
    assert L.zjai_conv1x1_weight_grad(h, px, 0, 1, 4, 4, 8, 8, tp, dw.data_ptr(), None, D) == 0
    eng.sync()
    assert not dw.any()
    # an arena too small for a call's scratch
    import zenjpegai_b200 as zj
    small = zj.Engine(0, arena_bytes=1 << 26)
    try:
        with pytest.raises(zj.ZjaiError) as e:
            small.tape_pack(np.zeros((64, 512, 512), np.float32))
        assert e.value.status == big
    finally:
        small.close()
