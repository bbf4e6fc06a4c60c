"""Layer calls on a caller's stream whose parameters come from work that the stream still holds: the
parameters that the host reads are those at their place in the stream."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import zenjpegai_b200 as zj
    e = zj.Engine(0, arena_bytes=1 << 28)
    yield e
    e.close()


CALLS = [lambda e, x, w, b, wt, ws: e.conv2d(x, w, b, pad=(1, 1)),
         lambda e, x, w, b, wt, ws: e.conv_transpose2d(x, wt, b),
         lambda e, x, w, b, wt, ws: e.conv2d_backward(x, w, 24, 40, pad=(1, 1)),
         lambda e, x, w, b, wt, ws: e.conv_transpose2d_backward(x, wt, 12, 20),
         lambda e, x, w, b, wt, ws: e.transformer_ffn(x, *ws)]


def test_parameters_made_on_the_stream(eng):
    torch.manual_seed(2)

    def made(*shape, std):
        return torch.randn(*shape, device="cuda") * std

    x = made(64, 24, 40, std=1.0)
    params = (made(64, 64, 3, 3, std=0.05), made(64, std=0.1), made(64, 64, 4, 4, std=0.05),
              (made(64, std=1.0), made(64, std=0.1), made(128, 64, std=0.1),
               made(128, 1, 3, 3, std=0.3), made(64, 64, std=0.1)))
    torch.cuda.synchronize()
    want = [call(eng, x, *params) for call in CALLS]
    torch.cuda.synchronize()

    def late(t, zero):
        return tuple(late(v, zero) for v in t) if isinstance(t, tuple) else t + zero

    stream = torch.cuda.Stream()
    eng.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            for k, call in enumerate(CALLS):
                # the parameters appear some milliseconds after the call is made
                noise = torch.randn(4096, 4096, device="cuda")
                for _ in range(12):
                    noise = noise @ noise / 64
                zero = (noise[0, 0] * 0).nan_to_num()
                got = call(eng, x, *late(params, zero))
                assert np.array_equal(got.cpu().numpy(), want[k].cpu().numpy()), k
    finally:
        torch.cuda.synchronize()
        eng.set_stream(None)
