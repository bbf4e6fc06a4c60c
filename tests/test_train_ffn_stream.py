"""The stream that a GatedFFN's engine works on, with a stand-in for the engine: torch's current one in
each pass, whichever that is, and the caller's own setting before and after."""

import types

import pytest
import torch


class FakeEngine:
    """Every layer call notes the stream it came on and gives maps of the right shape."""

    device, stream = 0, None

    def __init__(self):
        self.calls = []

    def set_stream(self, s):
        self.stream = s or None

    def __getattr__(self, name):
        def call(*args, **kw):
            self.calls.append((name, self.stream))
            if name == "tape_pack":
                return types.SimpleNamespace(v=args[0])
            if name == "tape_unpack":
                return args[0].v
            if name == "conv2d":
                return torch.zeros(args[1].shape[0], *args[0].shape[1:])
            if name == "depthwise3x3_elu_gate":
                return torch.zeros(args[0].shape[0] // 2, *args[0].shape[1:])
            if name == "conv2d_backward":
                c = args[0].shape[0] if kw.get("groups") else args[1].shape[1]
                return torch.zeros(c, *args[0].shape[1:])
            if name == "elu_gate_backward":
                return torch.zeros_like(args[1]), torch.zeros_like(args[2])
            if name == "gated_residual_norm":
                x = args[0]
                return x, x, {k: types.SimpleNamespace(v=x) for k in ("f", "y")}
            if name == "gated_residual_norm_backward":
                c = kw["scale"].shape
                return dict({"x": args[0], "f": args[0]}, **{k: torch.zeros(c) for k in (
                    "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")})
            if name == "conv1x1_weight_grad":
                return torch.zeros(args[0].shape[0], args[1].v.shape[0]), torch.zeros(args[0].shape[0])
            return args[0]  # depthwise3x3
        return call


@pytest.fixture
def current(monkeypatch):
    """torch's current stream, as a handle to set."""
    now = types.SimpleNamespace(cuda_stream=0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now)
    return now


@pytest.mark.parametrize("own", [None, 55])
def test_each_pass_on_the_current_stream(current, own):
    from zenjpegai_b200 import STREAM_LEGACY
    from zenjpegai_b200.train_ffn import GatedFFN
    e = FakeEngine()
    e.set_stream(own)
    current.cuda_stream = 11
    net = GatedFFN(e, 4, 6, 2, device="cpu")
    assert e.stream == own  # the engine's other users find it as it was
    x = torch.zeros(4, 3, 5)
    for forward, backward in ((0, 0), (77, 77), (77, 99), (0, 77)):
        current.cuda_stream, e.calls = forward, []
        net.forward(x)
        assert e.calls and {s for _, s in e.calls} == {forward or STREAM_LEGACY}
        assert e.stream == own
        current.cuda_stream, e.calls = backward, []
        net.backward(x, x)
        assert e.calls and {s for _, s in e.calls} == {backward or STREAM_LEGACY}
        assert e.stream == own


def test_left_as_it_was_after_an_error(current):
    from zenjpegai_b200.train_ffn import GatedFFN
    e = FakeEngine()
    net = GatedFFN(e, 4, 6, 1, device="cpu")
    e.set_stream(55)
    current.cuda_stream = 77
    with pytest.raises(AttributeError):
        net.forward(None)
    assert e.stream == 55
