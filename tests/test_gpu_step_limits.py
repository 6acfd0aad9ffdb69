"""apeiron_b200.step at the ends of its arguments: windows of any size, lengths and bounds that do
not fit, pages that no query sees any more."""
import numpy as np
import pytest

import step_ref as ref
from test_gpu_step import batch_of, check_attention, gpu, random_pages

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from apeiron_b200 import Backend
    from apeiron_b200.step import StepOps

    be = Backend(0)
    yield StepOps(be)
    be.close()


# ---- windows -------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 704, 703, 699])
@pytest.mark.parametrize("sinks", [0, 5, 2 ** 31 - 1])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [300, 700]), ([40, 9], [700, 50]),
                                            ([260], [700])])
def test_attention_wide_windows(ops, kind, window, sinks, q_lens, kv_lens):
    """Windows of all the keys, of all that the table has room for (704 of 16-token pages), and
    up to the type's end: one row, a block of rows and many, on each kernel."""
    check_attention(ops, q_lens, kv_lens, 14, 2, 64, 16, kind, window, sinks)


@pytest.mark.parametrize("kind", ["float32", "float16"])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (7, 0), (7, 3), (60, 0)])
@pytest.mark.parametrize("q_lens,kv_lens", [([3, 1], [1, 0]), ([200], [150]), ([30, 7], [20, 7])])
def test_attention_window_before_the_first_key(ops, kind, window, sinks, q_lens, kv_lens):
    """Queries that stand before token 0 under a window: zeros."""
    check_attention(ops, q_lens, kv_lens, 8, 2, 64, 16, kind, window, sinks)
