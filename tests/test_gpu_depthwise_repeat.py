"""The streaming depthwise kernel, time after time with the operands in the caches and not: a row's
reads and the copy that takes its place in shared memory must not depend on which comes first.

Tolerance as for the layers' other tests against f32: 1e-3 relative L2 (f16 storage)."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("c,h,w,gate", [(384, 128, 128, False), (1024, 128, 128, True),
                                        (128, 500, 333, False), (128, 501, 334, True)])
def test_same_bits(c, h, w, gate):
    import zenjpegai_b200 as zj
    eng = zj.Engine(0, arena_bytes=1 << 30)
    eng.set_stream(zj.STREAM_LEGACY)
    try:
        torch.manual_seed(c)
        x = torch.randn(c, h, w, device="cuda")
        wt = torch.randn(c, 1, 3, 3, device="cuda") * 0.3
        call = eng.depthwise3x3_elu_gate if gate else eng.depthwise3x3
        want = F.conv2d(x.double()[None], wt.double(), padding=1, groups=c)[0]
        if gate:
            want = F.elu(want[:c // 2]) * want[c // 2:]
        cold = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
        first = call(x, wt)
        assert float((first.double() - want).norm()) <= 1e-3 * float(want.norm())
        for i in range(30):
            if i % 2:
                cold.zero_()
            assert torch.equal(call(x, wt), first), i
    finally:
        torch.cuda.synchronize()
        eng.close()
