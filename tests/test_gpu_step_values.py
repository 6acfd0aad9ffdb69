"""apeiron_b200.step's values where the arithmetic is at its weakest, and forms that the operators
offer beside the usual ones, against tests/step_ref.py and 64 bits."""
import numpy as np
import pytest

import step_ref as ref
from test_gpu_step import gpu, norm_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from apeiron_b200 import Backend
    from apeiron_b200.step import StepOps

    be = Backend(0)
    yield StepOps(be)
    be.close()


# ---- norm ---------------------------------------------------------------------------------

@pytest.mark.parametrize("n,k", [(64, 1), (896, 3), (1500, 4), (4096, 2), (4096, 200), (8192, 160),
                                 (16000, 150), (40000, 3)])
@pytest.mark.parametrize("large", [40.0, 4099.7, 1e6])
def test_norm_with_dominant_channels(ops, n, k, large):
    """A large value behind small ones, at every place of a thread's four: the sum of squares keeps
    what f32 would lose.  Its error, some 2^-36 of it at most, turns the rounding of a y over with a
    probability of 2^-11; plain f32's, 2^-24 of it, of one in two."""
    import torch

    rng = np.random.default_rng(n + k)
    x = rng.standard_normal((k, n)).astype(np.float32)
    for r in range(k):
        x[r, (r % 4) + 4 * rng.integers(0, (n - 4) // 4, max(1, n // 300))] = large * rng.uniform(1, 2)
    w = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
    y = torch.empty(k, n, device="cuda")
    ops.add_rms_norm_quant(gpu(x), gpu(w), 1e-6, y=y)
    want = norm_ref(x, w.astype(np.float64), np.float64(np.float32(1e-6)))
    got = y.cpu().numpy()
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want))
    turned = (got != want.astype(np.float32)).sum()
    assert turned <= max(2, n * k * 2.0 ** -10)
