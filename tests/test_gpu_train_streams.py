"""Calls of one engine on several streams: they share its scratch, so each waits for the one before."""

import numpy as np
import pytest
import torch

import test_gpu_train as base
import train_reference as ref
from test_gpu_train import eng  # noqa: F401

pytestmark = pytest.mark.gpu


def test_streams_taken_in_turn(eng):  # noqa: F811
    """Weight gradients whose partial tiles lie in the engine's arena, and parameter sums likewise, on
    two streams of torch and the engine's own: the bits of calls made one after the other."""
    import zenjpegai_b200 as zj
    rng = np.random.default_rng(3)
    shape = (4, 64, 64, 64)
    one = base.dev(np.ones(64))
    douts = [base.dev(rng.standard_normal((4, 192, 64, 64))) for _ in range(3)]
    tapes = [eng.tape_pack(base.dev(rng.standard_normal(shape))) for _ in range(3)]
    dys = [base.dev(rng.standard_normal(shape)) for _ in range(3)]

    def work(i):
        g = eng.gated_residual_norm_backward(dys[i], dys[i - 1], y=tapes[i], pre=(one, one))
        return eng.conv1x1_weight_grad(douts[i], tapes[i]) + tuple(g[k] for k in sorted(g))

    want = []
    for i in range(3):
        want.append(work(i))
        torch.cuda.synchronize()
    x, d = ref.unpack(*(t.cpu().numpy() for t in (tapes[0].codes, tapes[0].exps))), base.f64(douts[0])
    ww, _ = ref.weight_grad(d, x)
    mw, _ = ref.weight_grad(np.abs(d), np.abs(x))
    assert (np.abs(base.f64(want[0][0]) - ww) <= base.SUM_TOL * mw).all()
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()]
    got = []
    try:
        for turn in range(60):
            i = turn % 3
            with torch.cuda.stream(streams[i]):
                eng.set_stream((None, zj.STREAM_LEGACY)[turn // 3 % 2] if i == 2
                               else streams[i].cuda_stream)
                got.append((i, work(i)))
    finally:
        torch.cuda.synchronize()
        eng.set_stream(None)
    for i, g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_stream_set_under_capture(eng):  # noqa: F811
    """A stream may be set and left while it is captured: no order is put between the two."""
    rng = np.random.default_rng(4)
    x = base.dev(rng.standard_normal((2, 16, 32, 32)))
    want = eng.tape_pack(x)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=stream):
            eng.set_stream(stream.cuda_stream)
            tape = eng.tape_pack(x)
            eng.set_stream(None)
    finally:
        eng.set_stream(None)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tape.codes, want.codes) and torch.equal(tape.exps, want.exps)
    assert torch.equal(eng.tape_pack(x).codes, want.codes)
    torch.cuda.synchronize()
    del graph
