"""The 64-bit definitions that the training operators are tested against, themselves checked: the
backward pass against central differences of the forward one, the tape format against its bounds,
and the Python side's refusals that need no GPU."""

import numpy as np
import pytest

import train_reference as ref


@pytest.mark.parametrize("gate_channels", [0, 1, 5])
@pytest.mark.parametrize("parts", ["", "p", "s", "n", "ps", "pn", "psn"])
def test_backward_against_differences(gate_channels, parts):
    rng = np.random.default_rng(len(parts) * 10 + gate_channels)
    n, c, h, w = 2, 5, 2, 3
    v = {"x": rng.standard_normal((n, c, h, w)), "f": rng.standard_normal((n, c, h, w))}
    if gate_channels:
        v["gate"] = rng.standard_normal((n, gate_channels, h, w))
    if "s" in parts:
        v["scale"] = rng.standard_normal(c)
    for k, on in (("post", "p" in parts), ("pre", "n" in parts)):
        if on:
            v[k + "_weight"], v[k + "_bias"] = rng.standard_normal(c), rng.standard_normal(c)
    dy, dz = rng.standard_normal((n, c, h, w)), rng.standard_normal((n, c, h, w))

    def kw(v):
        pair = lambda k: (v[k + "_weight"], v[k + "_bias"]) if k + "_weight" in v else None  # noqa: E731
        return {"post": pair("post"), "gate": v.get("gate"), "scale": v.get("scale"),
                "pre": pair("pre")}

    def loss(v):
        y, z = ref.residual(v["x"], v["f"], **kw(v))
        return (y * dy).sum() + ((z * dz).sum() if z is not None else 0.0)

    y, _ = ref.residual(v["x"], v["f"], **kw(v))
    got, _ = ref.residual_backward(dy, dz, v["f"], y, **kw(v))
    step = 1e-5
    for name, val in v.items():
        for at in range(min(val.size, 12)):
            i = at * 7 % val.size
            up = {k: a.copy() for k, a in v.items()}
            down = {k: a.copy() for k, a in v.items()}
            up[name].flat[i] += step
            down[name].flat[i] -= step
            want = (loss(up) - loss(down)) / (2 * step)
            # central differences: step^2 / 6 of the third derivative, and 1e-16 / step rounding
            assert abs(got[name].flat[i] - want) < 1e-6 * (1 + abs(want)), (name, i)


def test_tape_bounds():
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((1, 3, 5, 29)) * np.exp2(rng.integers(-30, 30, (1, 3, 5, 29))))
    x[0, 0, 0, 0] = 127.9  # saturates: a whole step off at most
    x[0, 1] = 0.0
    codes, exps = ref.pack(x.astype(np.float32))
    back = ref.unpack(codes, exps)
    v = ref.groups_of(x.astype(np.float32).astype(np.float64).reshape(1, 3, -1))
    err = np.abs(ref.groups_of(back.reshape(1, 3, -1)) - v)
    step = np.exp2(exps.astype(np.float64))[..., None]
    assert (err <= np.where(np.abs(v) > 127 * step, step, step / 2)).all()
    # a value stays below the next power of two above its group's largest: finite where x is
    top = np.exp2(np.floor(np.log2(np.maximum(np.abs(v).max(3), 2.0 ** -120))) + 1)
    assert (np.abs(ref.groups_of(back.reshape(1, 3, -1))).max(3) < top).all()
    assert not back[0, 1].any()
    x[0, 2, 0, 0] = np.inf
    codes, exps = ref.pack(x)
    assert exps[0, 2, 0] == 127 and np.isnan(ref.unpack(codes, exps)[0, 2].reshape(-1)[:32]).all()


class _NoEngine:
    device, handle, stream = 0, None, None


def test_refusals_before_the_library():
    import zenjpegai_b200 as zj
    from zenjpegai_b200 import tape as T
    e = _NoEngine()
    f32 = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    t = zj.Tape(np.zeros((4, 3, 5), np.int8), np.zeros((4, 1), np.int8))
    bad = [
        lambda: T.tape_pack(e, f32(4, 6, 5)[:, ::2]),                      # not contiguous
        lambda: T.tape_pack(e, np.zeros((4, 3, 5))),                       # float64
        lambda: T.tape_pack(e, f32(4, 15)),                                # not a map
        lambda: T.tape_unpack(e, zj.Tape(t.codes, np.zeros((4, 2), np.int8))),
        lambda: T.tape_unpack(e, zj.Tape(t.codes, np.zeros((4, 1), np.uint8))),
        lambda: T.tape_unpack(e, t, np.float64),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), f32(4, 5, 3)),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), np.zeros((4, 3, 5), np.float16)),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), f32(4, 3, 5), gate=f32(2, 3, 5)),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), f32(4, 3, 5), scale=f32(3)),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), f32(4, 3, 5), post=f32(4)),
        lambda: T.gated_residual_norm(e, f32(4, 3, 5), f32(4, 3, 5), tape=("q",)),
        lambda: T.gated_residual_norm_backward(e, f32(4, 3, 5), f=t, scale=f32(4), gate=f32(4, 3, 5)),
        lambda: T.gated_residual_norm_backward(e, f32(4, 3, 5), scale=f32(4)),
        lambda: T.gated_residual_norm_backward(e, f32(4, 3, 5), dz=f32(4, 3, 5)),
        lambda: T.gated_residual_norm_backward(e, f32(4, 3, 5), pre=(f32(4), f32(4)), y=t),
        lambda: T.conv1x1_weight_grad(e, f32(6, 3, 4), t),
        lambda: T.conv1x1_weight_grad(e, f32(6, 3, 5), f32(4, 3, 5)),
        lambda: T.conv1x1_weight_grad(e, f32(1, 6, 3, 5), t),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(zj.ZjaiError) as err:
            call()
        assert err.value.status == zj._lib.INVALID_ARGUMENT, i
