"""Timed cases of the training operators: 8-bit activation tapes, the gated residual norm and its
backward pass, and the weight gradient of a 1x1 projection from a tape.

`own = False` computes each operator in its plain form (elementary torch operations in 32 bits,
rounded once at the end); `own = True` makes the calls a user makes of `zenjpegai_b200.Engine`.

The operators, on maps [n, c, h, w] with P = h w positions per channel row:

* tape: groups of 32 consecutive positions of a row share the power of two
  2^e, e = clamp(floor(log2 max|x|) - 6, -126, 121); code = clamp(rint(x 2^-e), -127, 127); a group
  that holds an infinity or a NaN has e = 127 and stands for NaN.
* gated residual norm: y = x + scale sigmoid(gate) LN_post(f), z = LN_pre(y), the layer norms over
  the channels of a position (eps 1e-5).
* its backward pass, from dy and dz and the taped f, gate and y.
* weight gradient: dw = sum over pictures and positions of dout x^T from the taped x, db = sum dout.
"""

import math

import torch

own = False

EPS = 1e-5
GROUP = 32
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_TAPED = 1.0 + 1.0 / GROUP  # bytes of one taped element


# ---- cases -----------------------------------------------------------------------------------

def listed():
    return [
        # the map of one small region, its rows not a multiple of a group
        {"name": "tape region f32", "op": "tape", "dtype": "f32", "n": 1, "c": 64, "h": 33, "w": 29},
        # the gate map (2 x 512 hidden channels) of the 28 interior tiles of a 4K picture
        {"name": "tape ffn 4k f16", "op": "tape", "dtype": "f16", "n": 28, "c": 1024, "h": 128,
         "w": 128},
        # one position: what a residual step costs at the least
        {"name": "norm one position f32", "op": "norm", "dtype": "f32", "n": 1, "c": 128, "h": 1,
         "w": 1, "gate": "full", "tape": False},
        # a residual step of the luma network's transformer blocks (dim 128) on the 4K picture's
        # 28 interior tiles, taped for the backward pass
        {"name": "norm 4k f32 taped", "op": "norm", "dtype": "f32", "n": 28, "c": 128, "h": 128,
         "w": 128, "gate": "full", "tape": True},
        # three regions of odd size, one gate for all channels of a position
        {"name": "norm odd bf16", "op": "norm", "dtype": "bf16", "n": 3, "c": 160, "h": 67, "w": 45,
         "gate": "position", "tape": False},
        # the backward pass on a small region (chroma dim 64)
        {"name": "norm back small f32", "op": "norm_back", "dtype": "f32", "n": 1, "c": 64, "h": 16,
         "w": 16, "gate": "full", "tape": True},
        # the backward pass of the 4K residual step from its tape
        {"name": "norm back 4k f32", "op": "norm_back", "dtype": "f32", "n": 28, "c": 128, "h": 128,
         "w": 128, "gate": "full", "tape": True},
        # odd maps in half precision whose activations were kept as they are
        {"name": "norm back odd f16", "op": "norm_back", "dtype": "f16", "n": 4, "c": 192, "h": 135,
         "w": 61, "gate": "position", "tape": False},
        # a projection's weight gradient on one small region
        {"name": "wgrad small f32", "op": "wgrad", "dtype": "f32", "n": 1, "oc": 128, "c": 128,
         "h": 16, "w": 16},
        # the qkv projection (128 -> 384) of the 4K picture's tiles
        {"name": "wgrad qkv 4k f32", "op": "wgrad", "dtype": "f32", "n": 28, "oc": 384, "c": 128,
         "h": 128, "w": 128},
        # the feed-forward input projection (128 -> 1024) of the same tiles
        {"name": "wgrad ffn 4k bf16", "op": "wgrad", "dtype": "bf16", "n": 28, "oc": 1024, "c": 128,
         "h": 128, "w": 128},
        # an odd projection on two odd regions
        {"name": "wgrad odd f16", "op": "wgrad", "dtype": "f16", "n": 2, "oc": 200, "c": 72,
         "h": 101, "w": 77},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    case = {"op": rng.choice(["tape", "norm", "norm_back", "wgrad"]),
            "dtype": rng.choice(["f32", "f16", "bf16"]), "n": spread(1, 28)}
    if case["op"] == "wgrad":
        case["oc"] = spread(16, 1024)
        case["c"] = spread(16, 512)
    else:
        case["c"] = spread(16, 1024 if case["op"] == "tape" else 512)
    # half of the channel counts are the multiples of 16 that networks have
    if rng.random() < 0.5:
        case["c"] = max(16, case["c"] // 16 * 16)
        if "oc" in case:
            case["oc"] = max(16, case["oc"] // 16 * 16)
    case["h"], case["w"] = spread(1, 256), spread(1, 256)
    if rng.random() < 0.5:
        case["w"] = max(16, case["w"] // 16 * 16)
    if case["op"] in ("norm", "norm_back"):
        case["gate"] = rng.choice(["full", "position", "none"])
        case["tape"] = rng.random() < 0.6
    most = {"tape": 2.8e9, "norm": 2.1e9, "norm_back": 1.3e9, "wgrad": 1.0e9}[case["op"]]
    while work(case)["bytes"] > most or work(case)["flops"] > 1.2e11:
        if case["n"] > 1:
            case["n"] //= 2
        else:
            case["h"] = (case["h"] + 1) // 2
    return case


def work(case):
    n, c, p, s = case["n"], case["c"], case["h"] * case["w"], _SIZE[case["dtype"]]
    e = n * c * p
    if case["op"] == "tape":  # x read, codes written; codes read, x written
        return {"bytes": 2 * e * (s + _TAPED), "flops": 4 * e}
    if case["op"] == "wgrad":
        oc = case["oc"]
        return {"bytes": n * p * (oc * s + c * _TAPED) + 4 * oc * (c + 1),
                "flops": 2 * n * p * oc * c}
    gate = {"full": e, "position": n * p, "none": 0}[case["gate"]]
    if case["op"] == "norm":  # x, f, gate -> y, z; the tape of f, gate, y, z, read back as bf16
        b = 4 * e * s + gate * s + 20 * c
        if case["tape"]:
            b += (3 * e + gate) * (2 * _TAPED + 2)
        return {"bytes": b, "flops": 24 * e}
    kept = _TAPED if case["tape"] else s  # dy, dz and f, y, gate -> dx, df, dgate
    return {"bytes": 4 * e * s + 2 * e * kept + gate * (s + kept) + 40 * c, "flops": 50 * e}


# ---- inputs ----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    n, c, h, w = case["n"], case["c"], case["h"], case["w"]

    def randn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    def activation(channels):
        # channels of unlike spread, as a network's residual stream has them
        x = torch.randn(n, channels, h, w, generator=g, device="cuda", dtype=torch.float32)
        x *= torch.exp(0.7 * randn(1, channels, 1, 1))
        return x.add_(0.3 * randn(1, channels, 1, 1)).to(dt)

    st = {"case": case}
    if case["op"] == "tape":
        st["x"] = activation(c)
        return st
    if case["op"] == "wgrad":
        st["x"] = pack(activation(c))
        st["dout"] = randn(n, case["oc"], h, w, std=1e-2, dtype=dt)
        return st
    st["post"] = (1.0 + randn(c, std=0.1), randn(c, std=0.1))
    st["pre"] = (1.0 + randn(c, std=0.1), randn(c, std=0.1))
    st["scale"] = 0.5 + randn(c, std=0.1)
    gc = {"full": c, "position": 1, "none": 0}[case["gate"]]
    st["gate"] = randn(n, gc, h, w, std=1.5, dtype=dt) if gc else None
    st["f"] = activation(c)
    if case["op"] == "norm":
        st["x"] = activation(c)
        return st
    st["y"] = activation(c)
    st["dy"] = randn(n, c, h, w, std=1e-2, dtype=dt)
    st["dz"] = randn(n, c, h, w, std=1e-2, dtype=dt)
    if case["tape"]:
        st["f"], st["y"] = pack(st["f"]), pack(st["y"])
        st["gate"] = pack(st["gate"]) if gc else None
    return st


# ---- plain forms -----------------------------------------------------------------------------

def _pow2(e):
    """2^e of int32 exponents in -126..127, exactly."""
    return ((e + 127) << 23).view(torch.float32)


def pack(x):
    """(codes int8 [n, c, h, w], exps int8 [n, c, groups])."""
    n, c, h, w = x.shape
    p = h * w
    groups = -(-p // GROUP)
    v = torch.zeros(n, c, groups * GROUP, dtype=torch.float32, device=x.device)
    v[:, :, :p] = x.reshape(n, c, p)
    v = v.view(n, c, groups, GROUP)
    a = v.abs().amax(3)
    e = ((a.view(torch.int32) >> 23) - 133).clamp(-126, 121)
    fine = torch.isfinite(a)
    codes = torch.round(v * _pow2(-e)[..., None]).clamp(-127, 127)
    codes = torch.where(fine[..., None], codes, torch.zeros_like(codes)).to(torch.int8)
    codes = codes.view(n, c, groups * GROUP)[:, :, :p].reshape(n, c, h, w).contiguous()
    return codes, torch.where(fine, e, torch.full_like(e, 127)).to(torch.int8)


def unpack(taped):
    codes, exps = taped
    n, c, h, w = codes.shape
    p = h * w
    s = _pow2(exps.int().clamp(-126, 126))
    s = torch.where(exps == 127, torch.full_like(s, math.nan), s)
    s = s.repeat_interleave(GROUP, 2)[:, :, :p].reshape(n, c, h, w)
    return codes.float() * s


def _values(v):
    return unpack(v) if isinstance(v, tuple) else v.float()


def _normal(v):
    """(v - mean) / sigma over the channels, and 1 / sigma."""
    d = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * r, r


def _col(p):
    return p.view(1, -1, 1, 1)


def _plain_norm(st):
    x, f = st["x"].float(), st["f"].float()
    u = _normal(f)[0] * _col(st["post"][0]) + _col(st["post"][1])
    q = _col(st["scale"])
    if st["gate"] is not None:
        q = q * torch.sigmoid(st["gate"].float())
    y = x + q * u
    z = _normal(y)[0] * _col(st["pre"][0]) + _col(st["pre"][1])
    dt = st["x"].dtype
    out = {"y": y.to(dt), "z": z.to(dt)}
    if st["case"]["tape"]:
        for name, v in (("f", f), ("gate", st["gate"]), ("y", y), ("z", z)):
            if v is not None:
                out["tape_" + name] = unpack(pack(v)).to(torch.bfloat16)
    return out


def _plain_norm_back(st):
    dt = st["dy"].dtype
    dy, dz = st["dy"].float(), st["dz"].float()
    f, y = _values(st["f"]), _values(st["y"])
    yn, r2 = _normal(y)
    a = dz * _col(st["pre"][0])
    d = dy + (a - a.mean(1, keepdim=True) - yn * (a * yn).mean(1, keepdim=True)) * r2
    out = {"x": d.to(dt), "pre_weight": (dz * yn).sum((0, 2, 3)), "pre_bias": dz.sum((0, 2, 3))}
    fn, r1 = _normal(f)
    u = fn * _col(st["post"][0]) + _col(st["post"][1])
    du = d * _col(st["scale"])
    if st["gate"] is None:
        out["scale"] = (d * u).sum((0, 2, 3))
    else:
        sg = torch.sigmoid(_values(st["gate"]))
        out["scale"] = (d * u * sg).sum((0, 2, 3))
        dg = du * u * sg * (1.0 - sg)
        out["gate"] = (dg.sum(1, keepdim=True) if sg.shape[1] < u.shape[1] else dg).to(dt)
        du = du * sg
    out["post_weight"], out["post_bias"] = (du * fn).sum((0, 2, 3)), du.sum((0, 2, 3))
    a = du * _col(st["post"][0])
    df = (a - a.mean(1, keepdim=True) - fn * (a * fn).mean(1, keepdim=True)) * r1
    out["f"] = df.to(dt)
    return out


def _plain_wgrad(st):
    n, oc = st["dout"].shape[:2]
    d = st["dout"].float().reshape(n, oc, -1)
    x = unpack(st["x"]).reshape(n, st["case"]["c"], -1)
    return {"dw": torch.matmul(d, x.transpose(1, 2)).sum(0), "db": d.sum((0, 2))}


# ---- the framework's operators -----------------------------------------------------------------

_eng = None


def _engine():
    """The engine a program keeps, working on torch's default stream."""
    global _eng
    if _eng is None:
        import zenjpegai_b200 as zj
        _eng = zj.Engine(0, arena_bytes=1 << 28)
        _eng.set_stream(zj.STREAM_LEGACY)
    return _eng


def _kept(v):
    if not isinstance(v, tuple):
        return v
    from zenjpegai_b200 import Tape
    return Tape(*v)


def _own(st):
    eng, case = _engine(), st["case"]
    if case["op"] == "tape":
        return {"restored": eng.tape_unpack(eng.tape_pack(st["x"]), st["x"].dtype)}
    if case["op"] == "wgrad":
        dw, db = eng.conv1x1_weight_grad(st["dout"], _kept(st["x"]))
        return {"dw": dw, "db": db}
    if case["op"] == "norm":
        y, z, tapes = eng.gated_residual_norm(
            st["x"], st["f"], post=st["post"], gate=st["gate"], scale=st["scale"], pre=st["pre"],
            tape=("f", "gate", "y", "z") if case["tape"] else ())
        out = {"y": y, "z": z}
        for name, t in tapes.items():
            out["tape_" + name] = eng.tape_unpack(t, torch.bfloat16)
        return out
    return eng.gated_residual_norm_backward(
        st["dy"], st["dz"], f=_kept(st["f"]), y=_kept(st["y"]), post=st["post"],
        gate=_kept(st["gate"]), scale=st["scale"], pre=st["pre"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "tape":
        return {"restored": unpack(pack(state["x"])).to(state["x"].dtype)}
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_back":
        return _plain_norm_back(state)
    return _plain_wgrad(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _exact_taped(x):
    """What the tape of one picture's map [c, h, w] stands for, by the definition."""
    c, h, w = x.shape
    v = x.double().reshape(c, h * w)
    out = torch.empty_like(v)
    whole = h * w // GROUP * GROUP
    for lo, hi in ((0, whole), (whole, h * w)):  # the whole groups, and the short one
        if lo == hi:
            continue
        k = v[:, lo:hi].reshape(c, -1, min(GROUP, hi - lo))
        top = k.abs().amax(2, keepdim=True)
        e = (torch.frexp(top)[1] - 7).clamp(-126, 121)  # top = m 2^e, m in [1/2, 1)
        step = ((e.long() + 1023) << 52).view(torch.float64)
        k = torch.minimum((k / step).round().abs(), torch.full_like(k, 127.0)) * k.sign() * step
        out[:, lo:hi] = k.reshape(c, -1)
    return out.reshape(c, h, w)


def _exact_values(v, i):
    """Picture i of a kept map in 64 bits."""
    if not isinstance(v, tuple):
        return v[i].double()
    codes, exps = v[0][i], v[1][i]
    c, h, w = codes.shape
    at = torch.arange(h * w, device=codes.device) // GROUP
    e = exps.double()[:, at]
    s = torch.where(e == 127, torch.full_like(e, math.nan), torch.exp2(e))
    return codes.double() * s.reshape(c, h, w)


def _exact_stats(v):
    """1 / sigma and the normalised values of one picture [c, h, w]."""
    c = v.shape[0]
    mean = v.sum(0) / c
    sigma = (((v - mean) ** 2).sum(0) / c + EPS).sqrt()
    return sigma, (v - mean) / sigma


def exact(case, seed):
    st = prepare(case, seed)
    n = case["n"]
    if case["op"] == "tape":
        r = torch.empty(st["x"].shape, dtype=torch.float64, device="cuda")
        for i in range(n):
            r[i] = _exact_taped(st["x"][i])
        return {"restored": r}
    if case["op"] == "wgrad":
        dw = torch.zeros(case["oc"], case["c"], dtype=torch.float64, device="cuda")
        db = torch.zeros(case["oc"], dtype=torch.float64, device="cuda")
        for i in range(n):
            d = st["dout"][i].double().reshape(case["oc"], -1)
            dw += d @ _exact_values(st["x"], i).reshape(case["c"], -1).t()
            db += d.sum(1)
        return {"dw": dw, "db": db}
    w1, b1 = (p.double().view(-1, 1, 1) for p in st["post"])
    w2, b2 = (p.double().view(-1, 1, 1) for p in st["pre"])
    sc = st["scale"].double().view(-1, 1, 1)

    def gate_of(i):
        return 1.0 / (1.0 + torch.exp(-_exact_values(st["gate"], i))) if st["gate"] is not None else None

    if case["op"] == "norm":
        y = torch.empty(st["x"].shape, dtype=torch.float64, device="cuda")
        z = torch.empty_like(y)
        out = {"y": y, "z": z}
        if case["tape"]:
            # the tapes of y and z hold roundings of computed values: no value of their own
            out.update(tape_f=torch.empty_like(y), tape_y=None, tape_z=None)
            if st["gate"] is not None:
                out["tape_gate"] = torch.empty(st["gate"].shape, dtype=torch.float64, device="cuda")
        for i in range(n):
            u = _exact_stats(st["f"][i].double())[1] * w1 + b1
            sg = gate_of(i)
            y[i] = st["x"][i].double() + (sc * u if sg is None else sc * sg * u)
            z[i] = _exact_stats(y[i])[1] * w2 + b2
            for name in ("f", "gate"):
                if out.get("tape_" + name) is not None:
                    out["tape_" + name][i] = _exact_taped(st[name][i])
        return out
    big = torch.empty(n, case["c"], case["h"], case["w"], dtype=torch.float64, device="cuda")
    sums = [torch.zeros(case["c"], dtype=torch.float64, device="cuda") for _ in range(5)]
    out = {"x": big, "f": torch.empty_like(big), "scale": sums[0], "post_weight": sums[1],
           "post_bias": sums[2], "pre_weight": sums[3], "pre_bias": sums[4]}
    if st["gate"] is not None:
        gc = case["c"] if case["gate"] == "full" else 1
        out["gate"] = torch.empty(n, gc, case["h"], case["w"], dtype=torch.float64, device="cuda")
    for i in range(n):
        dz = st["dz"][i].double()
        s2, yn = _exact_stats(_exact_values(st["y"], i))
        t = dz * w2
        d = st["dy"][i].double() + (t - t.mean(0) - yn * (t * yn).mean(0)) / s2
        s1, fn = _exact_stats(_exact_values(st["f"], i))
        u = fn * w1 + b1
        sg = gate_of(i)
        one = torch.ones_like(u) if sg is None else sg.expand_as(u)
        du = d * sc * one
        if sg is not None:
            dg = d * sc * u * one * (1.0 - one)
            out["gate"][i] = dg.sum(0, keepdim=True) if case["gate"] == "position" else dg
        t = du * w1
        out["x"][i] = d
        out["f"][i] = (t - t.mean(0) - fn * (t * fn).mean(0)) / s1
        for k, v in enumerate((d * one * u, du * fn, du, dz * yn, dz)):
            sums[k] += v.sum((1, 2))
    return out
