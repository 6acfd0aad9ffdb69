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


@pytest.mark.parametrize("n", [1, 33, 896, 1537, 4096, 20000])
@pytest.mark.parametrize("k,extra", [(1, 0), (5, 0), (5, 3), (200, 4)])
def test_norm_values_in_f32(ops, n, k, extra):
    """The activation that the codes stand for, as f32: code * S to the bit, in rows apart."""
    import torch

    rng = np.random.default_rng(n + k)
    x = (rng.standard_normal((k, n)) * np.exp(2 * rng.standard_normal((k, 1)))).astype(np.float32)
    x[k // 2] = 0
    deq = torch.full((k, n + extra), 7.0, device="cuda")
    act = ops.add_rms_norm_quant(gpu(x), None, 1e-5)
    assert ops.add_rms_norm_quant(gpu(x), None, 1e-5, deq=deq[:, :n]) is None
    e = act.exps[:, : -(-n // 32)].cpu().numpy().astype(np.int64)
    s = np.where(e == 0xFF, 0.0, np.ldexp(1.0, e - 32)).repeat(32, 1)[:, :n]
    want = act.codes[:, :n].cpu().numpy() * s
    assert np.array_equal(deq[:, :n].cpu().numpy().astype(np.float64), want)
    assert (deq[:, n:] == 7.0).all()


# ---- sampler --------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(5, 40), (12, 5003), (12, 32003), (60, 33000), (9, 151936)])
def test_sample_filters_of_each_row(ops, rows, vocab):
    """A served batch: every row has filters and a temperature of its own, some none at all."""
    from test_gpu_step import check_sample

    rng = np.random.default_rng(rows + vocab)
    logits = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    logits[1::2, :: max(1, vocab // 60)] += 8
    pick = lambda *v: rng.choice(v, rows)  # noqa: E731
    check_sample(ops, logits, rng.random(rows), pad=3,
                 temperature=pick(0.0, 0.3, 1.0, 1.0, 2.5), top_k=pick(0, 1, 40, 40, 1000, 3000),
                 top_p=pick(1.0, 1.0, 0.1, 0.9, 0.97), min_p=pick(0.0, 0.0, 0.02, 0.3))


# ---- positions ------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,dim", [(5, 1, 64), (64, 8, 128), (12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("rot,layout", [(64, "half"), (64, "interleaved"), (24, "half"), (8, "half")])
def test_append_turns_q_in_place(ops, heads, kv_heads, dim, rot, layout):
    """q_out = q, in the fused rows of a projection: the bits of an output of its own."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    t = 200
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = torch.randn(t, (heads + 2 * kv_heads) * dim, device="cuda")
    batch = SeqBatch(torch.tensor([0, t], **i32), torch.tensor([t], **i32),
                     torch.arange(13, **i32)[None].contiguous(), t, t)
    cache = KV4Cache.empty(13, kv_heads, dim, 16)
    table = ops.rope_table(t, rot)

    def run(rows, q_out):
        q, k, v = (p.unflatten(1, (-1, dim)) for p in
                   rows.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        return ops.rope_kv4_append(q, k, v, table, cache, batch, rot_dim=rot, layout=layout,
                                   q_out=q if q_out else None)

    want = run(rows, False)
    for _ in range(5):
        copy = rows.clone()
        run(copy, True)
        assert torch.equal(copy[:, : heads * dim], want.flatten(1))
        assert torch.equal(copy[:, heads * dim:], rows[:, heads * dim:])
    q = rows[:, : heads * dim].unflatten(1, (heads, dim))
    k = torch.randn(t, kv_heads, dim, device="cuda")
    for other in (rows.view(torch.bfloat16)[:, : heads * dim],  # the same place, another type
                  rows.view(-1)[: t * heads * dim].view(t, -1)):  # or other rows
        with pytest.raises(ValueError):
            ops.rope_kv4_append(q, k, k, table, cache, batch, rot_dim=rot, layout=layout,
                                q_out=other.unflatten(1, (heads, dim)))
