"""A stack of gated feed-forward halves (`TransformerBlock::forward`, attention.rs:346-371, with a
residual scale, a gate and a post-norm on the branch) trained from 8-bit tapes: how the training
operators are used together.

A half with input x and its norm z:
    h = W_in . z + b_in, d = dw3x3(h), m = elu(d_1) . d_2, f = W_out . m + b_out
    y = x + scale . sigmoid(gate) . LN_post(f), z' = LN_pre(y)        (one gated_residual_norm)
Forward holds z, d, m, f and y in 8 bits: 1.03 bytes an element in place of 4. Backward reads them
there: the residual step's gradients from the tapes of f and y, the weights' from those of m and z.
The depthwise weights are fixed; everything else is trained.

Usage: python -m zenjpegai_b200.train_ffn [--dim C] [--hidden C] [--size S] [--depth N] [--steps N]
"""

import argparse
import contextlib

import torch

from . import STREAM_LEGACY, Engine


@contextlib.contextmanager
def _on_current_stream(engine):
    """The engine on torch's current stream, where its layers and torch's own kernels take turns; then
    on the one that it was set to before."""
    before = engine.stream
    engine.set_stream(torch.cuda.current_stream(engine.device).cuda_stream or STREAM_LEGACY)
    try:
        yield
    finally:
        engine.set_stream(before)


class GatedFFN:
    """`depth` halves on maps [dim, h, w]: parameters as float32 CUDA tensors in `params`, a list
    of dicts; `forward` keeps the tapes that `backward` reads. Each pass works on the stream that is
    torch's current one as it is called, and leaves the engine's stream as it was."""

    def __init__(self, engine, dim, hidden, depth, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(*shape, generator=g) * std).to(device)

        self.engine, self.dim, self.hidden = engine, dim, hidden
        self.tapes = []
        self.params = [{
            "w_in": normal(2 * hidden, dim, std=dim ** -0.5), "b_in": normal(2 * hidden, std=0.02),
            "w_out": normal(dim, hidden, std=hidden ** -0.5), "b_out": normal(dim, std=0.02),
            "post_weight": torch.ones(dim, device=device),
            "post_bias": torch.zeros(dim, device=device),
            "scale": torch.full((dim,), 0.5, device=device),
            "pre_weight": torch.ones(dim, device=device),
            "pre_bias": torch.zeros(dim, device=device),
        } for _ in range(depth)]
        self.w_dw = [normal(2 * hidden, 1, 3, 3, std=0.05) for _ in range(depth)]
        for w in self.w_dw:
            w[:, 0, 1, 1] += 1.0

    def _step(self, p):
        return {"post": (p["post_weight"], p["post_bias"]), "scale": p["scale"],
                "pre": (p["pre_weight"], p["pre_bias"])}

    def forward(self, x, gate=None):
        """x [dim, h, w] and the gate's logits, [1, h, w] or like x: the last half's (y, z)."""
        with _on_current_stream(self.engine):
            return self._forward(x, gate)

    def _forward(self, x, gate):
        e, z = self.engine, x
        self.tapes = []
        for p, w_dw in zip(self.params, self.w_dw):
            h = e.conv2d(z, p["w_in"][:, :, None, None], p["b_in"])
            d = e.depthwise3x3(h, w_dw)
            m = e.depthwise3x3_elu_gate(h, w_dw)
            f = e.conv2d(m, p["w_out"][:, :, None, None], p["b_out"])
            tapes = {"z": e.tape_pack(z), "d": e.tape_pack(d), "m": e.tape_pack(m)}
            x, z, more = e.gated_residual_norm(x, f, gate=gate, tape=("f", "gate", "y"),
                                               **self._step(p))
            self.tapes.append({**tapes, **more})
        return x, z

    def backward(self, dy, dz):
        """From the gradients of the last half's y and z: those of x and of the gate (None without
        one), and of each half's parameters."""
        with _on_current_stream(self.engine):
            return self._backward(dy, dz)

    def _backward(self, dy, dz):
        e, grads, dgate = self.engine, [], None
        for p, w_dw, t in zip(self.params[::-1], self.w_dw[::-1], self.tapes[::-1]):
            h, w = dy.shape[1:]
            g = e.gated_residual_norm_backward(dy, dz, f=t["f"], y=t["y"], gate=t.get("gate"),
                                               **self._step(p))
            gp = {k: g[k] for k in ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")}
            if "gate" in t:
                dgate = g["gate"] if dgate is None else dgate + g["gate"]
            gp["w_out"], gp["b_out"] = e.conv1x1_weight_grad(g["f"], t["m"])
            dm = e.conv2d_backward(g["f"], p["w_out"][:, :, None, None], h, w)
            d = e.tape_unpack(t["d"])
            dd = torch.cat(e.elu_gate_backward(dm, d[:self.hidden], d[self.hidden:]))
            dh = e.conv2d_backward(dd, w_dw, h, w, pad=(1, 1), groups=2 * self.hidden)
            gp["w_in"], gp["b_in"] = e.conv1x1_weight_grad(dh, t["z"])
            dz = e.conv2d_backward(dh, p["w_in"][:, :, None, None], h, w)
            dy = g["x"]
            grads.insert(0, gp)
        # the first half's z is its x
        return dy + dz, dgate, grads

    def tape_bytes(self):
        return sum(t.codes.numel() + t.exps.numel() for half in self.tapes for t in half.values())


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--size", type=int, default=128)
    ap.add_argument("--depth", type=int, default=2)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--rate", type=float, default=20.0)
    a = ap.parse_args()
    engine = Engine(0, arena_bytes=1 << 30)
    torch.manual_seed(1)
    x = torch.randn(a.dim, a.size, a.size, device="cuda")
    gate = torch.randn(1, a.size, a.size, device="cuda")
    want, _ = GatedFFN(engine, a.dim, a.hidden, a.depth, seed=7).forward(x, gate)
    net = GatedFFN(engine, a.dim, a.hidden, a.depth)
    for step in range(a.steps):
        y, _ = net.forward(x, gate)
        diff = y - want
        loss = float((diff * diff).mean()) / 2
        _, _, grads = net.backward(diff / diff.numel(), torch.zeros_like(diff))
        for p, g in zip(net.params, grads):
            for k in p:
                p[k] -= a.rate * g[k]
        print("step %d  loss %.5f  tapes %.1f MB" % (step, loss, net.tape_bytes() / 1e6))
    engine.close()


if __name__ == "__main__":
    main()
