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


@pytest.mark.parametrize("rows,vocab", [(1, 1000), (1, 16000), (3, 40000), (40, 32003)])
def test_sampler_logits_from_the_call_before(ops, rows, vocab):
    """The logits are what the norm before has written."""
    import torch

    rng = np.random.default_rng(vocab)
    sources = gpu(rng.standard_normal((30, rows, vocab)).astype(np.float32))
    logits = torch.zeros(rows, vocab, device="cuda")
    u = torch.rand(30, rows, device="cuda")
    token = torch.empty(30, rows, dtype=torch.int32, device="cuda")
    top_k = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for i in range(30):
        ops.add_rms_norm_quant(sources[i], None, 1e-6, y=logits)
        ops.sample(logits, u[i], top_k=top_k, token=token[i])
    torch.cuda.synchronize()
    for i in range(30):
        ops.add_rms_norm_quant(sources[i], None, 1e-6, y=logits)
        torch.cuda.synchronize()
        assert torch.equal(ops.sample(logits, u[i], top_k=top_k), token[i])


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("nq", [1, 16, 200])
def test_attention_over_pages_of_the_call_before(ops, kind, nq):
    """The keys and values are those that the append before has written over others."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(nq)
    i32 = dict(dtype=torch.int32, device="cuda")
    dt = getattr(torch, kind)
    batch = SeqBatch(torch.tensor([0, nq], **i32), torch.tensor([nq], **i32),
                     torch.arange(-(-nq // 16), **i32)[None].contiguous(), nq, nq)
    cache = KV4Cache.empty(-(-nq // 16), 2, 64, 16)
    qkv = gpu(rng.standard_normal((30, nq, 12, 64)).astype(np.float32))
    table = ops.rope_table(nq, 64)
    q = torch.empty(nq, 8, 64, device="cuda", dtype=dt)
    out = torch.empty(30, nq, 8, 64, device="cuda", dtype=dt)
    torch.cuda.synchronize()

    def step(i, out, wait):
        ops.rope_kv4_append(qkv[i, :, :8], qkv[i, :, 8:10], qkv[i, :, 10:], table, cache, batch,
                            rot_dim=64, q_out=q)
        if wait:
            torch.cuda.synchronize()
        ops.attn_kv4(q, cache, batch, 0.125, out=out)

    for i in range(30):
        step(i, out[i], False)
    torch.cuda.synchronize()
    want = torch.empty_like(q)
    for i in range(30):
        step(i, want, True)
        assert torch.equal(out[i], want)


def test_attention_in_a_context_just_opened(ops):
    """The first call of a context, at once and on a stream that waits for no other: its keys are
    split over the GPU and joined through counters that start at zero."""
    import torch
    from apeiron_b200 import Backend
    from apeiron_b200.step import KV4Cache, SeqBatch, StepOps

    i32 = dict(dtype=torch.int32, device="cuda")
    cache = KV4Cache(torch.randint(0, 100, (200, 1, 1152), dtype=torch.uint8, device="cuda"), 1, 64, 16)
    batch = SeqBatch(torch.tensor([0, 1], **i32), torch.tensor([3200], **i32),
                     torch.arange(200, **i32)[None].contiguous(), 1, 1)
    q = torch.randn(1, 4, 64, device="cuda")
    want = ops.attn_kv4(q, cache, batch, 0.1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        be = Backend(0)
        out = StepOps(be).attn_kv4(q, cache, batch, 0.1, out=torch.empty_like(q),
                                   stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(out, want)
        be.close()


@pytest.mark.parametrize("call", ["norm", "table", "append", "attention", "sample"])
def test_outputs_on_another_stream(ops, call):
    """What a call on a given stream allocates is not memory that the current stream, which it does
    not wait for, still has to write: here late, over blocks of the same sizes that are free again."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(0)
    t = 300
    i32 = dict(dtype=torch.int32, device="cuda")
    x = gpu(rng.standard_normal((t, 12, 64)).astype(np.float32))
    cache = KV4Cache.empty(20, 2, 64, 16)
    batch = SeqBatch(torch.tensor([0, t], **i32), torch.tensor([t], **i32),
                     torch.arange(20, **i32)[None].contiguous(), t, t)
    table = ops.rope_table(t, 64)
    u = torch.rand(t, device="cuda")
    side = torch.cuda.Stream()

    def run(stream):
        if call == "norm":
            act = ops.add_rms_norm_quant(x.flatten(1), None, 1e-6, stream=stream)
            return act.codes, act.exps, act.descs
        if call == "table":
            return (ops.rope_table(t, 64, stream=stream),)
        if call == "append":
            return (ops.rope_kv4_append(x[:, :8], x[:, 8:10], x[:, 10:], table, cache, batch,
                                        rot_dim=64, stream=stream),)
        if call == "attention":
            return (ops.attn_kv4(x[:, :8], cache, batch, 0.1, stream=stream),)
        return (ops.sample(x.flatten(1), u, stream=stream),)

    ops.rope_kv4_append(None, x[:, 8:10], x[:, 10:], table, cache, batch, rot_dim=64)
    torch.cuda.synchronize()
    want = [w.clone() for w in run(None)]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    late = [torch.empty_like(w) for w in want for _ in range(3)]
    torch.cuda._sleep(100_000_000)
    for m in late:
        m.fill_(1)
    del m, late
    got = run(side.cuda_stream)
    side.synchronize()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("call", ["norm", "append", "attention", "prompt", "sample"])
def test_captured_behind_a_copy(ops, call):
    """A captured call behind a copy from the host reads what the copy brings, at every replay."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(1)
    t = 120
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = SeqBatch(torch.tensor([0, t], **i32), torch.tensor([t], **i32),
                     torch.arange(8, **i32)[None].contiguous(), t, t)
    cache = KV4Cache.empty(8, 2, 64, 16)
    table, u = ops.rope_table(t, 64), torch.rand(t, device="cuda")
    kv = gpu(rng.standard_normal((t, 2, 64)).astype(np.float32))
    ops.rope_kv4_append(None, kv, kv, table, cache, batch, rot_dim=64)
    dt = torch.bfloat16 if call == "prompt" else torch.float32
    x, y = (torch.zeros(t, 8, 64, dtype=dt, device="cuda") for _ in range(2))
    token = torch.zeros(t, **i32)
    fresh = torch.from_numpy(rng.standard_normal((6, t, 8, 64)).astype(np.float32)).to(dt)
    host = torch.empty(t, 8, 64, dtype=dt).pin_memory()

    def run():
        if call == "norm":
            ops.add_rms_norm_quant(x.flatten(1), None, 1e-6, y=y.view(t, 512))
        elif call == "append":
            ops.rope_kv4_append(x, kv, kv, table, cache, batch, rot_dim=64, q_out=y)
        elif call == "sample":
            ops.sample(x.flatten(1), u, token=token)
        else:
            ops.attn_kv4(x, cache, batch, 0.1, out=y)

    run()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        x.copy_(host, non_blocking=True)
        run()
    for v in fresh:
        host.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = (y.clone(), token.clone())
        x.copy_(v)
        run()
        assert torch.equal(got[0], y) and torch.equal(got[1], token)


def test_default_and_current_stream_by_handle(ops):
    """The handles of the default stream (0) and of the current one serve as streams too."""
    import torch

    x = torch.randn(6, 500, device="cuda")
    u = torch.rand(6, device="cuda")
    want = ops.sample(x, u)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert torch.equal(ops.sample(x, u, stream=0), want)
    assert torch.equal(ops.sample(x, u, stream=torch.cuda.current_stream().cuda_stream), want)
    with torch.cuda.stream(side):
        got = ops.sample(x, u, stream=side.cuda_stream)
        act = ops.add_rms_norm_quant(x, None, 1e-6, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(act.codes, ops.add_rms_norm_quant(x, None, 1e-6).codes)
