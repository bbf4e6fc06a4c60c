"""The weight gradient's bounded waits run out: with a limit of one SM cycle no role waits for anything
that is not there yet (the last products alone take hundreds), so every call gives up, says so in the
status word, and leaves the context as it was for the next one."""

import numpy as np
import pytest
import torch

import test_gpu_train as base
import train_reference as ref
from test_gpu_train import eng  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,oc,c,h,w", [(4, 256, 128, 64, 64), (2, 130, 40, 33, 65), (1, 16, 16, 1, 1)])
@pytest.mark.parametrize("dtype", list(base.DT))
def test_waits_run_out(eng, n, oc, c, h, w, dtype):  # noqa: F811
    import zenjpegai_b200 as zj
    rng = np.random.default_rng(oc)
    codes, exps = ref.pack(rng.standard_normal((n, c, h, w)))
    d = base.dev(rng.standard_normal((n, oc, h, w)) * 1e-2, dtype)
    tape = base.the_tape(codes, exps)
    want = eng.conv1x1_weight_grad(d, tape)
    torch.cuda.synchronize()
    for _ in range(10):
        eng.set_wait_limit(1)
        try:
            eng.conv1x1_weight_grad(d, tape)
            with pytest.raises(zj.ZjaiError) as err:
                eng.sync()
        finally:
            eng.set_wait_limit(0)
        assert err.value.status == 8  # ZJAI_DEVICE_TIMEOUT
        got = eng.conv1x1_weight_grad(d, tape)
        eng.sync()  # the status word was cleared
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_host_call_reports_it(eng):  # noqa: F811
    import zenjpegai_b200 as zj
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 64, 32, 32)).astype(np.float32)
    tape = eng.tape_pack(x)
    want = eng.conv1x1_weight_grad(x, tape)
    eng.set_wait_limit(1)
    try:
        with pytest.raises(zj.ZjaiError) as err:
            eng.conv1x1_weight_grad(x, tape)
    finally:
        eng.set_wait_limit(0)
    assert err.value.status == 8
    got = eng.conv1x1_weight_grad(x, tape)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_a_limit_that_suffices(eng):  # noqa: F811
    """Fifty milliseconds' limit changes nothing."""
    torch.manual_seed(0)
    d, x = torch.randn(28, 384, 64, 64, device="cuda"), torch.randn(28, 128, 64, 64, device="cuda")
    tape = eng.tape_pack(x)
    want = eng.conv1x1_weight_grad(d, tape)
    eng.set_wait_limit(100_000_000)
    try:
        got = eng.conv1x1_weight_grad(d, tape)
        eng.sync()
    finally:
        eng.set_wait_limit(0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
