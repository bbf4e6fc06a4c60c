"""The training operators' definitions in 64 bits (numpy), for the tests: the tape format, the gated
residual norm with its backward pass, and the weight gradient of a 1x1 convolution. Maps are
[n, c, h, w]."""

import numpy as np

EPS = 1e-5
GROUP = 32


def groups_of(v):
    """v [n, c, p] in groups [n, c, groups, 32], zeros behind a short last one."""
    n, c, p = v.shape
    g = -(-p // GROUP)
    out = np.zeros((n, c, g * GROUP), v.dtype)
    out[:, :, :p] = v
    return out.reshape(n, c, g, GROUP)


def pack(x):
    n, c, h, w = x.shape
    v = groups_of(x.astype(np.float64).reshape(n, c, h * w))
    top = np.abs(v).max(3)
    fine = np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(fine & (top > 0), np.floor(np.log2(np.where(fine & (top > 0), top, 1.0))), -200)
    # log2 may round up to the next integer just below a power of two
    e = np.where(fine & (top > 0) & (np.exp2(np.clip(e, -1000, 1000)) > top), e - 1, e)
    e = np.clip(e - 6, -126, 121)
    codes = np.clip(np.rint(np.where(fine[..., None], v, 0.0) * np.exp2(-e)[..., None]), -127, 127)
    codes = codes.reshape(n, c, -1)[:, :, :h * w].reshape(x.shape).astype(np.int8)
    return codes, np.where(fine, e, 127).astype(np.int8)


def unpack(codes, exps):
    n, c, h, w = codes.shape
    e = exps.astype(np.float64)
    s = np.where(e == 127, np.nan, np.exp2(np.maximum(e, -126)))
    s = np.repeat(s, GROUP, axis=2)[:, :, :h * w].reshape(codes.shape)
    return codes.astype(np.float64) * s


def layer_norm(v):
    m = v.mean(1, keepdims=True)
    sigma = np.sqrt(((v - m) ** 2).mean(1, keepdims=True) + EPS)
    return (v - m) / sigma, sigma


def col(p):
    return np.asarray(p, np.float64).reshape(1, -1, 1, 1)


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-g))


def residual(x, f, post=None, gate=None, scale=None, pre=None):
    u = f if post is None else layer_norm(f)[0] * col(post[0]) + col(post[1])
    if gate is not None:
        u = u * sigmoid(gate)
    if scale is not None:
        u = u * col(scale)
    y = x + u
    z = None if pre is None else layer_norm(y)[0] * col(pre[0]) + col(pre[1])
    return y, z


def ln_vjp(d, vn, sigma, weight):
    """Input gradient of LN(v) weight + bias."""
    a = d * col(weight)
    return (a - a.mean(1, keepdims=True) - vn * (a * vn).mean(1, keepdims=True)) / sigma


def residual_backward(dy, dz, f, y, post=None, gate=None, scale=None, pre=None):
    """Gradients, and for each the magnitude that its rounding errors are in proportion to: the
    formula again with the magnitudes of all that it adds and subtracts (the normalised values and
    the norms' gradients are differences, which may cancel)."""
    def magnitude(v, sigma):
        return (np.abs(v) + np.abs(v).mean(1, keepdims=True)) / sigma

    def ln_magnitude(dm, vm, sigma, weight):
        a = dm * np.abs(col(weight))
        return (a + a.mean(1, keepdims=True) + vm * (a * vm).mean(1, keepdims=True)) / sigma

    d, out, mag = np.array(dy, np.float64), {}, {}
    dm = np.abs(d)

    def total(name, terms, magnitudes):
        out[name], mag[name] = terms.sum((0, 2, 3)), magnitudes.sum((0, 2, 3))

    if pre is not None:
        yn, s2 = layer_norm(y)
        ym = magnitude(y, s2)
        d = d + ln_vjp(dz, yn, s2, pre[0])
        dm = dm + ln_magnitude(np.abs(dz), ym, s2, pre[0])
        total("pre_weight", dz * yn, np.abs(dz) * ym)
        total("pre_bias", np.array(dz, np.float64), np.abs(dz))
    out["x"], mag["x"] = d, dm
    u, um = f, np.abs(f)
    if post is not None:
        fn, s1 = layer_norm(f)
        fm = magnitude(f, s1)
        u = fn * col(post[0]) + col(post[1])
        um = fm * np.abs(col(post[0])) + np.abs(col(post[1]))
    sg = np.ones_like(d) if gate is None else sigmoid(gate)
    sc = np.ones_like(d) if scale is None else col(scale)
    if scale is not None:
        total("scale", d * sg * u, dm * sg * um)
    if gate is not None:
        dg, gm = d * sc * u * sg * (1.0 - sg), dm * np.abs(sc) * um * sg * (1.0 - sg)
        if gate.shape[1] != dg.shape[1]:
            dg, gm = dg.sum(1, keepdims=True), gm.sum(1, keepdims=True)
        out["gate"], mag["gate"] = dg, gm
    du, dum = d * sc * sg, dm * np.abs(sc) * sg
    out["f"], mag["f"] = du, dum
    if post is not None:
        out["f"] = ln_vjp(du, fn, s1, post[0])
        mag["f"] = ln_magnitude(dum, fm, s1, post[0])
        total("post_weight", du * fn, dum * fm)
        total("post_bias", du, dum)
    return out, mag


def weight_grad(dout, x):
    d = dout.reshape(dout.shape[0], dout.shape[1], -1)
    v = x.reshape(x.shape[0], x.shape[1], -1)
    return np.einsum("nop,ncp->oc", d, v, optimize=True), d.sum((0, 2))
