"""A GatedFFN under torch streams other than the one it was made under, on an engine that has a stream
of its own: the bits of the same passes on the default stream, with inputs that arrive late."""

import pytest
import torch

from test_gpu_train_ffn import eng  # noqa: F401

pytestmark = pytest.mark.gpu


def everything(y, z, dx, dgate, grads):
    return [y, z, dx, dgate] + [g[k] for g in grads for k in sorted(g)]


def test_passes_under_other_streams(eng):  # noqa: F811
    from zenjpegai_b200.train_ffn import GatedFFN
    torch.manual_seed(1)
    x, gate = torch.randn(32, 40, 56, device="cuda"), torch.randn(1, 40, 56, device="cuda")
    dy, dz = torch.randn(32, 40, 56, device="cuda"), torch.randn(32, 40, 56, device="cuda")
    net = GatedFFN(eng, 32, 64, 2, seed=2)
    assert eng.stream is None

    def passes():
        y, z = net.forward(x + late, gate + late)
        return everything(y, z, *net.backward(dy + late, dz + late))

    late = torch.zeros((), device="cuda")
    want = passes()
    torch.cuda.synchronize()
    for _ in range(8):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            # what the inputs are made from is there some milliseconds after the calls
            noise = torch.randn(4096, 4096, device="cuda")
            for _ in range(8):
                noise = noise @ noise / 64
            late = (noise[0, 0] * 0).nan_to_num()
            got = passes()
        stream.synchronize()
        assert eng.stream is None
        assert all(torch.equal(a, b) for a, b in zip(got, want))
