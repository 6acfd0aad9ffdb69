"""Tokens from a decoder that never leaves the GPU: random weights, the whole step on the device.

    python examples/decode_step.py [--batch B] [--tokens N] [--layers L]

Each step of a Qwen2.5-0.5B-shaped model (hidden 896, 14 query and 2 KV heads of 64, FFN 4864)
runs, per layer: residual add + RMS norm into the 8-bit activation, the exact q/k/v projections,
rotary positions with the append to a 4-bit paged KV cache, attention over the cache, the exact
output projection, the second norm, gate/up, SwiGLU + quant_act, down; then the final norm, the
head and the sampler.  After one eager step the rest replay as a CUDA graph.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from apeiron_b200 import Backend, Q8_0, synth  # noqa: E402
from apeiron_b200._abi import CARRIER_F32  # noqa: E402
from apeiron_b200.step import DeviceAct, KV4Cache, SeqBatch, StepOps  # noqa: E402


class Linear:
    """A Q8_0 projection with random weights: device activations in, f32 (or Q32.32) out."""

    def __init__(self, ops, n_out, n_in, seed):
        self.ops, self.n_out, self.n_in = ops, n_out, n_in
        self.t = ops.backend.upload(Q8_0, synth.payload(Q8_0, n_out, n_in, seed), n_out, n_in)

    def __call__(self, act, out, status):
        q32, f32 = (out, None) if out.dtype is torch.int64 else (None, out)
        rc = self.ops.lib.apx_matmat_async(
            self.ops.ctx, self.t.handle, self.n_out, self.n_in, act.k, act.codes.data_ptr(),
            act.exps.data_ptr(), act.descs.data_ptr(), q32.data_ptr() if q32 is not None else None,
            f32.data_ptr() if f32 is not None else None, status.data_ptr(),
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0, rc


class Decoder:
    """``step(tokens)`` appends one token per request and draws the next ones."""

    def __init__(self, ops, *, hidden=896, heads=14, kv_heads=2, dim=64, ffn=4864, layers=24,
                 vocab=151936, batch=1, context=512, page=64, rope_base=1e6, seed=0):
        self.ops, self.dim, self.batch = ops, dim, batch
        dev = ops.device
        rng = np.random.default_rng(seed)
        f32 = dict(dtype=torch.float32, device=dev)

        def vector(n):
            return torch.from_numpy((1 + 0.1 * rng.standard_normal(n)).astype(np.float32)).to(dev)

        self.layers = []
        pages = -(-context // page)
        for i in range(layers):
            s = 100 * (seed + i)
            self.layers.append({
                "norm1": vector(hidden), "norm2": vector(hidden),
                "q": Linear(ops, heads * dim, hidden, s + 1),
                "k": Linear(ops, kv_heads * dim, hidden, s + 2),
                "v": Linear(ops, kv_heads * dim, hidden, s + 3),
                "o": Linear(ops, hidden, heads * dim, s + 4),
                "gate": Linear(ops, ffn, hidden, s + 5), "up": Linear(ops, ffn, hidden, s + 6),
                "down": Linear(ops, hidden, ffn, s + 7),
                "cache": KV4Cache.empty(batch * pages, kv_heads, dim, page, dev)})
        self.norm = vector(hidden)
        self.head = Linear(ops, vocab, hidden, 99)
        self.embed = torch.from_numpy(rng.standard_normal((vocab, hidden)).astype(np.float32)).to(dev)
        self.rope = ops.rope_table(context, dim, rope_base)
        # what a step writes: kept, so that its addresses do not change (and a graph can hold them)
        self.token = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)  # cached tokens
        table = torch.arange(batch * pages, dtype=torch.int32, device=dev).reshape(batch, pages)
        cu = torch.arange(batch + 1, dtype=torch.int32, device=dev)
        self.seqs = SeqBatch(cu, self.lens, table, batch, 1)
        self.x = torch.empty(batch, hidden, **f32)
        self.y = torch.empty(batch, hidden, **f32)
        self.act = DeviceAct.empty(ops, batch, hidden)
        self.act_o = DeviceAct.empty(ops, batch, heads * dim)
        self.act_h = DeviceAct.empty(ops, batch, ffn)
        for a in (self.act_o, self.act_h):
            a.codes.zero_()
        self.qkv = [torch.empty(batch, h, dim, **f32) for h in (heads, kv_heads, kv_heads)]
        self.q = torch.empty(batch, heads, dim, **f32)
        self.attn = torch.empty(batch, heads, dim, **f32)
        self.gate_up = [torch.empty(batch, ffn, dtype=torch.int64, device=dev) for _ in range(2)]
        self.logits = torch.empty(batch, vocab, **f32)
        self.u = torch.empty(batch, **f32)
        self.status = torch.empty(9, batch, 2, dtype=torch.int64, device=dev)
        self.step_status = ops.new_status()
        self.refused = torch.zeros((), dtype=torch.bool, device=dev)
        self.sampling = {}

    def _layer(self, w, add):
        ops, lib, st = self.ops, self.ops.lib, self.status
        stream = torch.cuda.current_stream().cuda_stream
        b = self.batch
        st.fill_(-1)
        ops.add_rms_norm_quant(self.x, w["norm1"], 1e-6, add=add, resid=self.x if add is not None
                               else None, act=self.act)
        for i, n in enumerate("qkv"):
            w[n](self.act, self.qkv[i], st[i])
        ops.rope_kv4_append(*self.qkv, self.rope, w["cache"], self.seqs, rot_dim=self.dim,
                            q_out=self.q, status=self.step_status)
        ops.attn_kv4(self.q, w["cache"], self.seqs, self.dim ** -0.5, out=self.attn,
                     status=self.step_status)
        o = self.act_o
        assert lib.apx_quant_f32_cols_async(ops.ctx, self.attn.data_ptr(), o.n, b,
                                            o.codes.data_ptr(), o.exps.data_ptr(),
                                            o.descs.data_ptr(), stream) == 0
        w["o"](o, self.y, st[3])
        ops.add_rms_norm_quant(self.x, w["norm2"], 1e-6, add=self.y, resid=self.x, act=self.act)
        for i, n in enumerate(("gate", "up")):
            w[n](self.act, self.gate_up[i], st[4 + i])
        h = self.act_h
        assert lib.apx_swiglu_quant_cols_async(
            ops.ctx, self.gate_up[0].data_ptr(), self.gate_up[1].data_ptr(), h.n, b, CARRIER_F32,
            None, h.codes.data_ptr(), h.exps.data_ptr(), h.descs.data_ptr(), st[6].data_ptr(),
            stream) == 0
        w["down"](h, self.y, st[7])
        self.refused |= (st != -1).any()

    def step(self):
        """One token of every request: from ``token`` and ``u`` to ``logits`` and ``token``."""
        self.lens += 1
        torch.index_select(self.embed, 0, self.token, out=self.x)
        for i, w in enumerate(self.layers):
            self._layer(w, self.y if i else None)
        self.ops.add_rms_norm_quant(self.x, self.norm, 1e-6, add=self.y, resid=self.x,
                                    act=self.act)
        self.status.fill_(-1)
        self.head(self.act, self.logits, self.status[8])
        self.refused |= (self.status != -1).any()
        self.ops.sample(self.logits, self.u, token=self.token, **self.sampling)

    def check(self):
        """Waits; raises where a step refused."""
        got = StepOps.check_status(self.step_status)
        if got is not None or bool(self.refused.item()):
            raise RuntimeError(f"a step refused: {got}")


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--layers", type=int, default=24)
    args = ap.parse_args()
    ops = StepOps(Backend(0))
    d = Decoder(ops, layers=args.layers, batch=args.batch, context=args.tokens + 8)
    rows = torch.ones(args.batch, device=ops.device)
    d.sampling = dict(temperature=0.8 * rows, top_k=(50 * rows).int(), top_p=0.95 * rows)
    d.token.copy_(torch.arange(1, args.batch + 1, dtype=torch.int32))
    gen = torch.Generator(device=ops.device)
    gen.manual_seed(1)
    out = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.rand(args.batch, generator=gen, device=ops.device, out=d.u)
        d.step()
        d.check()
        out.append(d.token.tolist())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            d.step()
        begin = time.perf_counter()
        for _ in range(args.tokens - 1):
            torch.rand(args.batch, generator=gen, device=ops.device, out=d.u)
            graph.replay()
            out.append(d.token.tolist())
        side.synchronize()
    took = time.perf_counter() - begin
    d.check()
    print(f"{args.batch} x {args.tokens} tokens, {1e3 * took / max(1, args.tokens - 1):.3f} ms a "
          f"step; request 0: {[t[0] for t in out][:16]}")


if __name__ == "__main__":
    main()
