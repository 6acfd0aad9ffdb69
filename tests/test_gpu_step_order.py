"""Calls of apeiron_b200.step behind one another on a stream: each reads what the call before it
wrote, whichever of its inputs that is, although their kernels may start while it still runs."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from apeiron_b200 import Backend
    from apeiron_b200.step import StepOps

    be = Backend(0)
    yield StepOps(be)
    be.close()


def gpu(a):
    import torch

    return torch.from_numpy(np.array(a, order="C")).cuda()


@pytest.mark.parametrize("n,rows", [(896, 1), (896, 400), (2048, 3), (4096, 2), (8192, 5)])
@pytest.mark.parametrize("before", [1, 150])
def test_norm_weights_from_the_call_before(ops, n, rows, before):
    """The weights are the last row that the norm before has written; the same bits as with weights
    that were there all along."""
    import torch

    rng = np.random.default_rng(n + before)
    x = gpu(rng.standard_normal((rows, n)).astype(np.float32))
    sources = gpu(rng.standard_normal((40, before, n)).astype(np.float32))
    y = torch.zeros(before, n, device="cuda")
    out = torch.empty(40, rows, n, device="cuda")
    torch.cuda.synchronize()
    for i in range(40):
        ops.add_rms_norm_quant(sources[i], None, 1e-6, y=y)
        ops.add_rms_norm_quant(x, y[-1], 1e-6, y=out[i])
    torch.cuda.synchronize()
    want = torch.empty(rows, n, device="cuda")
    for i in range(40):
        ops.add_rms_norm_quant(sources[i], None, 1e-6, y=y)
        torch.cuda.synchronize()
        weights = y[-1].clone()
        torch.cuda.synchronize()
        ops.add_rms_norm_quant(x, weights, 1e-6, y=want)
        assert torch.equal(out[i], want)
