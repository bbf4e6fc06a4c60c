"""The training operators on buffers that start anywhere: maps one element, codes and exponents one to
three bytes off their allocations' alignment, and tapes cut out of a batch. The checks and tolerances
are those of test_gpu_train.py; where the maps' rows start anywhere anyway, a buffer's place changes
no bit."""

import numpy as np
import pytest
import torch

import test_gpu_train as base
import train_reference as ref
from test_gpu_train import eng  # noqa: F401

pytestmark = pytest.mark.gpu

STEPS = [((3, 33, 5, 9), "full", "psn"), ((2, 64, 16, 16), "full", "psn"), ((1, 257, 5, 7), "full", "psn"),
         ((1, 160, 7, 13), "one", "psn"), ((1, 96, 3, 50), "none", "pn"), ((2, 1, 4, 11), "one", "ps"),
         ((9, 48, 12, 11), "full", "n"), ((1, 2100, 1, 5), "full", "psn"), ((1, 16, 67, 61), "full", "psn")]


def moved(t, by):
    """The same contiguous tensor, `by` elements behind its allocation's start."""
    buf = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    v = buf[by:].view(t.shape)
    v.copy_(t)
    return v


def moved_tape(t, codes, exps):
    import zenjpegai_b200 as zj
    return zj.Tape(moved(t.codes, codes), moved(t.exps, exps))


def step(shape, gate, parts, dtype):
    """Gradients in, what was kept (values and tapes), parameters, and how to check the results."""
    rng = np.random.default_rng(sum(shape) + len(parts))
    v, kw = base.step_case(rng, shape, base.gate_channels(gate, shape[1]), parts)
    dk = base.on_device(kw, dtype)
    dy = base.dev(rng.standard_normal(shape) * 1e-2, dtype)
    dz = base.dev(rng.standard_normal(shape) * 1e-2, dtype) if "n" in parts else None
    kept = {"f": base.dev(v["f"], dtype), "y": base.dev(v["x"], dtype)}
    if dk["gate"] is not None:
        kept["gate"] = dk["gate"]
    rk = base.as_f64(dk)
    dk.pop("gate")

    def check(got, held):
        r = dict(rk, gate=held.get("gate"))
        want, mag = ref.residual_backward(base.f64(dy), base.f64(dz) if dz is not None else None,
                                          held["f"], held["y"], **r)
        assert set(got) == set(want)
        for k in got:
            end = base.END[dtype] if k in ("x", "f", "gate") else 0.0
            small = 2.0 ** -25 if end and dtype == "f16" else 0.0
            err = np.abs(base.f64(got[k]) - want[k])
            assert (err <= base.SUM_TOL * mag[k] + end * np.abs(want[k]) + small).all(), k

    return dy, dz, kept, dk, check


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in b)


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype", list(base.DT))
def test_backward_from_moved_tapes(eng, shape, gate, parts, dtype):  # noqa: F811
    dy, dz, kept, dk, check = step(shape, gate, parts, dtype)
    packed = {k: ref.pack(base.f64(t)) for k, t in kept.items()}
    held = {k: ref.unpack(*t) for k, t in packed.items()}
    tapes = {k: base.the_tape(*t) for k, t in packed.items()}
    first = eng.gated_residual_norm_backward(dy, dz, **tapes, **dk)
    check(first, held)
    anywhere = shape[2] * shape[3] % 4 != 0
    # (codes, exponents) of f, y and the gate
    for by in ([(0, 1)] * 3, [(0, 2)] * 3, [(0, 3)] * 3, [(1, 0)] * 3, [(2, 0)] * 3, [(3, 2)] * 3,
               [(0, 1), (0, 2), (0, 3)], [(2, 3), (0, 0), (1, 1)]):
        at = {k: moved_tape(t, *by[i]) for i, (k, t) in enumerate(tapes.items())}
        got = eng.gated_residual_norm_backward(dy, dz, **at, **dk)
        check(got, held)
        assert not anywhere or same(got, first), by
    got = eng.gated_residual_norm_backward(moved(dy, 1), moved(dz, 1) if dz is not None else None,
                                           **tapes, **dk)
    check(got, held)
    assert not anywhere or same(got, first)


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype", list(base.DT))
def test_backward_from_moved_maps(eng, shape, gate, parts, dtype):  # noqa: F811
    dy, dz, kept, dk, check = step(shape, gate, parts, dtype)
    held = {k: base.f64(t) for k, t in kept.items()}
    first = eng.gated_residual_norm_backward(dy, dz, **kept, **dk)
    check(first, held)
    anywhere = shape[2] * shape[3] % 4 != 0
    for by in (1, 2, 3):
        got = eng.gated_residual_norm_backward(
            moved(dy, by), moved(dz, 1) if dz is not None else None,
            **{k: moved(t, by) for k, t in kept.items()}, **dk)
        check(got, held)
        assert not anywhere or same(got, first), by


@pytest.mark.parametrize("c,h,w", [(33, 5, 9), (33, 2, 5), (7, 4, 8), (5, 12, 20)])
def test_pictures_of_a_taped_batch(eng, c, h, w):  # noqa: F811
    """Each picture's part of a batch's tapes, wherever it begins, is a tape."""
    import zenjpegai_b200 as zj
    rng = np.random.default_rng(c + h)
    maps = {k: base.dev(rng.standard_normal((6, c, h, w))) for k in ("f", "y", "gate")}
    dy, dz = (base.dev(rng.standard_normal((6, c, h, w)) * 1e-2) for _ in range(2))
    ones = np.ones(c), np.zeros(c)
    one = tuple(map(base.dev, ones))
    kw = {"post": one, "pre": one, "scale": one[0]}
    tapes = {k: eng.tape_pack(t) for k, t in maps.items()}
    dout = base.dev(rng.standard_normal((6, 24, h, w)))
    for i in range(6):
        cut = {k: zj.Tape(t.codes[i], t.exps[i]) for k, t in tapes.items()}
        own = {k: zj.Tape(t.codes[i].clone(), t.exps[i].clone()) for k, t in tapes.items()}
        held = {k: base.f64(eng.tape_unpack(t))[None] for k, t in own.items()}
        want, mag = ref.residual_backward(base.f64(dy[i])[None], base.f64(dz[i])[None], held["f"],
                                          held["y"], post=ones, gate=held["gate"], scale=ones[0],
                                          pre=ones)
        for tape in (cut, own):
            got = eng.gated_residual_norm_backward(dy[i], dz[i], **tape, **kw)
            assert set(got) == set(want)
            for k in got:
                err = np.abs(base.f64(got[k]).reshape(want[k].shape) - want[k])
                assert (err <= base.SUM_TOL * mag[k]).all(), k
        assert torch.equal(eng.tape_unpack(cut["f"]), eng.tape_unpack(own["f"]))
        got, want = (eng.conv1x1_weight_grad(dout[i].clone(), t["y"]) for t in (cut, own))
        x, d = base.f64(eng.tape_unpack(own["y"]))[None], base.f64(dout[i])[None]
        ww, wb = ref.weight_grad(d, x)
        mw, mb = ref.weight_grad(np.abs(d), np.abs(x))
        for dw, db in (got, want):
            assert (np.abs(base.f64(dw) - ww) <= base.SUM_TOL * mw).all()
            assert (np.abs(base.f64(db) - wb) <= base.SUM_TOL * mb).all()


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("dtype", list(base.DT))
def test_moved_exponents_elsewhere(eng, by, dtype):  # noqa: F811
    """Unpacking and the weight gradient take exponents from any byte on."""
    rng = np.random.default_rng(by)
    for n, c, h, w in ((2, 40, 16, 16), (3, 33, 7, 13)):
        tape = eng.tape_pack(base.dev(rng.standard_normal((n, c, h, w))))
        at = moved_tape(tape, 0, by)
        assert torch.equal(eng.tape_unpack(at, base.DT[dtype]), eng.tape_unpack(tape, base.DT[dtype]))
        d = base.dev(rng.standard_normal((n, 24, h, w)), dtype)
        got, want = eng.conv1x1_weight_grad(d, at), eng.conv1x1_weight_grad(d, tape)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
