"""The steps between the projections together, as examples/decode_step.py runs them: a small
decoder with its whole step on the device, against the same step in numpy (f64 where the step is
f32; the 8-bit activations, 4-bit cache and whole-number sampling as they are defined)."""
import os
import sys

import numpy as np
import pytest

import step_ref as ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "examples"))

pytestmark = pytest.mark.gpu

SIZE = dict(hidden=256, heads=4, kv_heads=2, dim=64, ffn=512, layers=2, vocab=1003, context=48,
            page=16, rope_base=1e4)


@pytest.fixture(scope="module")
def ops():
    from apeiron_b200 import Backend
    from apeiron_b200.step import StepOps

    be = Backend(0)
    yield StepOps(be)
    be.close()


def run(ops, batch, steps, graph=False, **sampling):
    import torch
    from decode_step import Decoder

    d = Decoder(ops, batch=batch, **SIZE)
    rows = torch.ones(batch, device="cuda")
    d.sampling = {k: (v * rows).int() if k == "top_k" else v * rows for k, v in sampling.items()}
    d.token.copy_(torch.arange(3, 3 + batch, dtype=torch.int32))
    got = []
    u = np.random.default_rng(4).random((steps, batch)).astype(np.float32)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = None
        for i in range(steps):
            d.u.copy_(torch.from_numpy(u[i]))
            if graph and i == 1:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    d.step()
            if g is None:
                d.step()
            else:
                g.replay()
            got.append((d.token.tolist(), d.logits.clone()))
        side.synchronize()
    d.check()
    return d, got, u


def weights(t, n_out, n_in):
    """The f64 matrix of a Q8_0 payload."""
    b = t.reshape(n_out, -1, 34)
    return (b[:, :, :2].copy().view(np.float16).astype(np.float64)
            * b[:, :, 2:].view(np.int8)).reshape(n_out, -1)[:, :n_in]


def eight(y):
    """The values of y's 8-bit activation."""
    from apeiron_b200 import synth

    c, e = synth.quant_act_np(synth.f32_to_q32(y.astype(np.float32)))
    s = np.where(e == 0xFF, 0.0, np.ldexp(1.0, e.astype(int) - 32))
    return c * s.repeat(32)[: c.size]


def numpy_step(d, state, token, pos):
    """Logits of one request's step; state: per layer the values of its cached K and V."""
    from apeiron_b200 import synth

    def linear(n_out, n_in, seed, x):
        return (weights(synth.payload(8, n_out, n_in, seed), n_out, n_in) @ x).astype(np.float32)

    def norm(x, w):
        x = x.astype(np.float64)
        return (x / np.sqrt((x * x).mean() + 1e-6) * w.cpu().numpy().astype(np.float64))

    s = SIZE
    h, kv, dim = s["heads"], s["kv_heads"], s["dim"]
    cs = d.rope[pos].cpu().numpy()
    x = d.embed[token].cpu().numpy()
    for i, w in enumerate(d.layers):
        a = eight(norm(x, w["norm1"]))
        seed = 100 * i
        q = linear(h * dim, s["hidden"], seed + 1, a).reshape(h, dim)
        k = linear(kv * dim, s["hidden"], seed + 2, a).reshape(kv, dim)
        v = linear(kv * dim, s["hidden"], seed + 3, a).reshape(kv, dim)
        q = ref.rotate(q, cs, dim, "half").astype(np.float64)
        state[i][0].append(ref.four_bits(ref.rotate(k, cs, dim, "half")).astype(np.float64))
        state[i][1].append(ref.four_bits(v).astype(np.float64))
        kk, vv = np.array(state[i][0]), np.array(state[i][1])
        o = np.empty((h, dim))
        for j in range(h):
            p = kk[:, j // (h // kv)] @ q[j] * dim ** -0.5
            p = np.exp(p - p.max())
            o[j] = p / p.sum() @ vv[:, j // (h // kv)]
        x = x + linear(s["hidden"], h * dim, seed + 4, eight(o.ravel()))
        a = eight(norm(x, w["norm2"]))
        g, u = (linear(s["ffn"], s["hidden"], seed + 5 + j, a).astype(np.float64) for j in (0, 1))
        x = x + linear(s["hidden"], s["ffn"], seed + 7, eight(g / (1 + np.exp(-g)) * u))
    return linear(s["vocab"], s["hidden"], 99, eight(norm(x, d.norm)))


@pytest.mark.parametrize("batch", [1, 3])
def test_decoder_matches_numpy(ops, batch):
    """Every step's logits to 2 % of their size: a value at a rounding boundary of the 8- or 4-bit
    grids may fall to the other side on either arithmetic (one step of 1/127 or 1/8 of a group),
    nothing else differs by more than f32 roundings.  The tokens are the sampler's on the logits."""
    d, got, u = run(ops, batch, 20, temperature=0.9, top_k=40, top_p=0.9)
    states = [[([], []) for _ in d.layers] for _ in range(batch)]
    tokens = list(range(3, 3 + batch))
    for i, (drawn, logits) in enumerate(got):
        x = logits.cpu().numpy()
        for r in range(batch):
            want = numpy_step(d, states[r], tokens[r], i)
            assert np.linalg.norm(x[r] - want) <= 0.02 * np.linalg.norm(want)
            assert drawn[r] == ref.sample(x[r], u[i, r], 0.9, 40, 0.9)[0]
        tokens = drawn


def test_graph_replays_the_same_steps(ops):
    plain = run(ops, 2, 24, top_k=20)[1]
    graph = run(ops, 2, 24, graph=True, top_k=20)[1]
    assert [t for t, _ in plain] == [t for t, _ in graph]
    assert all((a == b).all() for (_, a), (_, b) in zip(plain, graph))
