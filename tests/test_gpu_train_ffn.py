"""The stack of gated feed-forward halves trained from 8-bit tapes (zenjpegai_b200/train_ffn.py)
against the same stack in 64-bit torch with autograd.

Tolerance, by derivation: a taped value is off by at most half a step, 2^-7 of its group's largest
power of two, uniformly: 2^-7 / sqrt(3) of it, and of a normal map's values (a third of their group's
largest in the mean square) about 1.4 % in relative L2. A half's gradients see five taped maps once
each, the first half's also the second's: the square root of ten times 1.4 % is 4.5 %, doubled for
what is taken more than once within a half (LN's statistics and its normalised map, both factors of
the gate). The convolutions' 1e-3 vanish beside it."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

GRAD_TOL = 0.09


@pytest.fixture(scope="module")
def eng():
    import zenjpegai_b200 as zj
    e = zj.Engine(0, arena_bytes=1 << 28)
    yield e
    e.close()


def plain(net, leaves, x, gate):
    import torch.nn.functional as F

    def norm(v, w, b):
        return F.layer_norm(v.permute(1, 2, 0), (v.shape[0],), w, b, 1e-5).permute(2, 0, 1)

    z = x
    for p, w_dw in zip(leaves, net.w_dw):
        h = F.conv2d(z[None], p["w_in"][:, :, None, None], p["b_in"])
        d = F.conv2d(h, w_dw.double(), padding=1, groups=h.shape[1])[0]
        m = F.elu(d[:net.hidden]) * d[net.hidden:]
        f = F.conv2d(m[None], p["w_out"][:, :, None, None], p["b_out"])[0]
        q = p["scale"][:, None, None]
        if gate is not None:
            q = q * torch.sigmoid(gate)
        x = x + q * norm(f, p["post_weight"], p["post_bias"])
        z = norm(x, p["pre_weight"], p["pre_bias"])
    return x, z


@pytest.mark.parametrize("dim,hidden,h,w,gates", [(32, 64, 24, 40, 0), (48, 40, 17, 31, 1),
                                                  (32, 48, 16, 33, 32)])
def test_gradients(eng, dim, hidden, h, w, gates):
    from zenjpegai_b200.train_ffn import GatedFFN
    torch.manual_seed(dim)
    net = GatedFFN(eng, dim, hidden, 2, seed=3)
    x = torch.randn(dim, h, w, device="cuda")
    gate = torch.randn(gates, h, w, device="cuda") if gates else None
    dy, dz = torch.randn(dim, h, w, device="cuda"), torch.randn(dim, h, w, device="cuda")
    y, z = net.forward(x, gate)
    dx, dgate, grads = net.backward(dy, dz)

    leaves = [{k: v.double().requires_grad_() for k, v in p.items()} for p in net.params]
    x64 = x.double().requires_grad_()
    g64 = gate.double().requires_grad_() if gates else None
    y64, z64 = plain(net, leaves, x64, g64)
    (y64 * dy.double() + z64 * dz.double()).sum().backward()

    def off(got, want):
        return float((got.double() - want).norm() / want.norm())

    assert off(y, y64.detach()) < 5e-3 and off(z, z64.detach()) < 5e-3  # no tape on the way
    assert off(dx, x64.grad) < GRAD_TOL
    assert (dgate is None) == (gate is None)
    if gates:
        assert off(dgate, g64.grad) < GRAD_TOL
    for got, want in zip(grads, leaves):
        assert got.keys() == want.keys()
        for k in got:
            assert off(got[k], want[k].grad) < GRAD_TOL, k


def test_it_learns_in_a_quarter_of_the_memory(eng):
    from zenjpegai_b200.train_ffn import GatedFFN
    torch.manual_seed(5)
    x = torch.randn(32, 32, 32, device="cuda")
    want, _ = GatedFFN(eng, 32, 64, 2, seed=9).forward(x)
    net = GatedFFN(eng, 32, 64, 2)
    losses = []
    for _ in range(12):
        y, _ = net.forward(x)
        diff = y - want
        losses.append(float((diff * diff).mean()))
        _, _, grads = net.backward(diff / 1024, torch.zeros_like(diff))
        for p, g in zip(net.params, grads):
            for k in p:
                p[k] -= 0.2 * g[k]
    assert losses[-1] < 0.8 * losses[0], losses
    values = 2 * 32 * 32 * (32 + 128 + 64 + 32 + 32)  # z, d, m, f, y of each half
    assert net.tape_bytes() == values * 33 // 32
