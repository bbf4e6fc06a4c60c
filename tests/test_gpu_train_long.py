"""The training operators where a block takes several tiles, runs of groups end inside rows and
pictures, and channels are spread over a cluster's blocks: the checks of test_gpu_train.py, with its
tolerances, on longer maps."""

import pytest
import torch

import test_gpu_train as base
from test_gpu_train import eng  # noqa: F401

pytestmark = pytest.mark.gpu

STEPS = [((9, 130, 37, 41), "full", "psn"), ((20, 24, 64, 64), "one", "psn"),
         ((2, 512, 64, 96), "full", "psn"), ((3, 768, 31, 33), "full", "psn"),
         ((1, 1024, 64, 65), "none", "pn"), ((1, 2048, 8, 160), "one", "psn"),
         ((1, 2049, 6, 30), "full", "psn"), ((40, 1, 40, 40), "full", "s")]


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_residual_norm(eng, shape, gate, parts, dtype):  # noqa: F811
    base.test_residual_norm(eng, shape, gate, parts, dtype)


@pytest.mark.parametrize("shape,gate,parts", STEPS)
@pytest.mark.parametrize("dtype,taped", [("f32", True), ("f32", False), ("bf16", True),
                                         ("bf16", False)])
def test_residual_norm_backward(eng, shape, gate, parts, dtype, taped):  # noqa: F811
    base.test_residual_norm_backward(eng, shape, gate, parts, dtype, taped)


@pytest.mark.parametrize("shape", [(3, 40, 129, 127), (1, 5000, 1, 2), (2, 3000, 1, 1),
                                   (1, 700, 1, 33), (4, 333, 1, 35), (2, 64, 100, 100)])
@pytest.mark.parametrize("dtype", list(base.DT))
@pytest.mark.parametrize("off", [False, True])
def test_tape_round_trip(eng, shape, dtype, off):  # noqa: F811
    base.test_tape_round_trip(eng, shape, dtype, off)


@pytest.mark.parametrize("n,oc,c,h,w", [(6, 130, 24, 45, 91), (2, 40, 140, 127, 129),
                                        (9, 256, 128, 64, 64)])
@pytest.mark.parametrize("dtype", list(base.DT))
@pytest.mark.parametrize("off", [False, True])
def test_weight_grad(eng, n, oc, c, h, w, dtype, off):  # noqa: F811
    base.test_weight_grad(eng, n, oc, c, h, w, dtype, off)


@pytest.mark.parametrize("n,oc,c,h,w", [(28, 384, 128, 64, 64), (12, 200, 128, 64, 96),
                                        (4, 256, 100, 63, 65)])
@pytest.mark.parametrize("dtype", list(base.DT))
def test_weight_grad_many_times(eng, n, oc, c, h, w, dtype):  # noqa: F811
    """The same bits every time, with the operands in the caches and not: what a chunk's reads and
    the next one's copies share must not depend on which comes first."""
    torch.manual_seed(n)
    d = (torch.randn(n, oc, h, w, device="cuda") * 1e-2).to(base.DT[dtype])
    tape = eng.tape_pack(torch.randn(n, c, h, w, device="cuda"))
    x, d64 = eng.tape_unpack(tape).double().reshape(n, c, -1), d.double().reshape(n, oc, -1)
    want = torch.bmm(d64, x.transpose(1, 2)).sum(0)
    most = torch.bmm(d64.abs(), x.abs().transpose(1, 2)).sum(0)
    cold = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(60):
        if i % 2:
            cold.zero_()
        dw, db = eng.conv1x1_weight_grad(d, tape)
        assert ((dw.double() - want).abs() <= base.SUM_TOL * most).all(), i
        assert ((db.double() - d64.sum((0, 2))).abs() <= base.SUM_TOL * d64.abs().sum((0, 2))).all(), i
        if first is None:
            first = dw, db
        assert torch.equal(dw, first[0]) and torch.equal(db, first[1]), i
