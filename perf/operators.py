"""The operators between the projections of a language model's step, as timed cases.

Four operators carry a token from one projection to the next and from the head's logits to a
token: the residual add + RMS norm that writes a projection's 8-bit activation, rotary positions
with the append to a paged 4-bit KV cache, attention over that cache, and the sampler.  `run`
computes each of them either in plain torch operations (32-bit arithmetic, rounded once at the end)
or, with `own` set, through apeiron_b200's entry points.  `exact` computes them in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TILE = 16          # tokens of one cache tile
GROUP = 32         # lanes that share a scale, in the cache and in an 8-bit activation
WEIGHT_ONE = 2.0 ** 31  # the sampler's integer weight of the most likely token


# ---- cases --------------------------------------------------------------------------------


def listed():
    return [
        # one decoded token of a 0.5B model: the smallest call, all latency
        {"name": "norm_decode_896", "op": "norm", "tokens": 1, "n": 896, "add": True},
        # a 512-token prefill of a 70B model's residual stream
        {"name": "norm_prefill_8192", "op": "norm", "tokens": 512, "n": 8192, "add": True},
        # one token for each of 32 requests, 1.5B shape (12 query heads, 2 KV heads)
        {"name": "rope_decode_b32", "op": "rope", "batch": 32, "q_min": 1, "q_max": 1,
         "kv_min": 1, "kv_max": 4000, "heads": 12, "kv_heads": 2, "dim": 128, "page": 64,
         "rot": 128, "layout": "half", "type": "bf16"},
        # a 512-token prefill of a 70B shape, interleaved pairs on half of each head
        {"name": "rope_prefill_512", "op": "rope", "batch": 1, "q_min": 512, "q_max": 512,
         "kv_min": 512, "kv_max": 512, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "rot": 64, "layout": "interleaved", "type": "f32"},
        # one request, one token, a short context, 0.5B shape: latency
        {"name": "attn_decode_b1", "op": "attn", "batch": 1, "q_min": 1, "q_max": 1,
         "kv_min": 777, "kv_max": 777, "heads": 14, "kv_heads": 2, "dim": 64, "page": 16,
         "window": 0, "sinks": 0, "type": "f32"},
        # a serving batch of ragged contexts, 70B shape: the cache's bytes decide
        {"name": "attn_decode_b64", "op": "attn", "batch": 64, "q_min": 1, "q_max": 1,
         "kv_min": 100, "kv_max": 4096, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "type": "bf16"},
        # one long context: the work has to be split along it
        {"name": "attn_decode_128k", "op": "attn", "batch": 1, "q_min": 1, "q_max": 1,
         "kv_min": 131001, "kv_max": 131001, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "type": "f32"},
        # two prompts, 1.5B shape, causal: matrix products on the tensor cores
        {"name": "attn_prefill_2k", "op": "attn", "batch": 2, "q_min": 1500, "q_max": 2048,
         "kv_min": 2048, "kv_max": 2500, "heads": 12, "kv_heads": 2, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "type": "bf16"},
        # a chunk of a prompt in 32-bit numbers, 0.5B shape, with a sliding window and sinks
        {"name": "attn_chunk_window", "op": "attn", "batch": 3, "q_min": 200, "q_max": 512,
         "kv_min": 1500, "kv_max": 2100, "heads": 14, "kv_heads": 2, "dim": 64, "page": 32,
         "window": 700, "sinks": 4, "type": "f32"},
        # one request's next token: the head's 151936 logits, all latency
        {"name": "sample_b1", "op": "sample", "rows": 1, "vocab": 151936, "top_k": 50,
         "top_p": 0.9, "min_p": 0.0},
        # a serving batch, nucleus and min-p without top-k
        {"name": "sample_b64", "op": "sample", "rows": 64, "vocab": 151936, "top_k": 0,
         "top_p": 0.95, "min_p": 0.02},
        # a small odd vocabulary, every filter at work
        {"name": "sample_b7_odd", "op": "sample", "rows": 7, "vocab": 32003, "top_k": 1000,
         "top_p": 0.98, "min_p": 0.001},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = max(lo, min(hi, v))
    return v - (v == 3072)


def draw(rng):
    op = rng.choice(["norm", "rope", "attn", "attn", "attn", "sample"])
    if op == "norm":
        n = _spread(rng, 64, 8192)
        return {"op": op, "n": n, "add": rng.random() < 0.7, "tokens": _spread(rng, 1, 512)}
    if op == "sample":
        return {"op": op, "rows": _spread(rng, 1, 64), "vocab": _spread(rng, 1000, 151936),
                "top_k": rng.choice([0, _spread(rng, 1, 2000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)])}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (12, 2, 128), (64, 8, 128), (16, 16, 64),
                                       (32, 4, 128), (8, 1, 128), (20, 4, 64)])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "rope":
        q = rng.choice([1, 1, _spread(rng, 2, 400)])
        b = _spread(rng, 1, 64 if q == 1 else max(1, 1000 // q))
        hi = _spread(rng, q + 1, q + 4000)
        return {**c, "batch": b, "q_min": max(1, q // 2), "q_max": q, "kv_min": q, "kv_max": hi,
                "rot": rng.choice([dim, dim // 2, dim // 4]),
                "layout": rng.choice(["half", "interleaved"])}
    window = rng.choice([0, 0, _spread(rng, 16, 2000)])
    c = {**c, "window": window, "sinks": rng.choice([0, 4, 17]) if window else 0}
    if rng.random() < 0.6:  # decode: the cache's bytes of all requests stay below the listed ones'
        b = _spread(rng, 1, 64)
        most = max(64, min(120000, 200000 * 8 // (b * kv_heads)))
        hi = _spread(rng, 40, most)
        return {**c, "batch": b, "q_min": 1, "q_max": rng.choice([1, 1, 1, 3]),
                "kv_min": rng.choice([0, hi // 4, hi]), "kv_max": hi}
    q = _spread(rng, 20, 1500)
    b = rng.choice([1, 2, 3])
    hi = _spread(rng, q + 1, q + 1500)
    if q * hi * b * heads > 30_000_000 * (2 if c["type"] != "f32" else 1):
        b, q = 1, min(q, 600)
    return {**c, "batch": b, "q_min": max(1, q // 2), "q_max": q, "kv_min": max(q, hi // 2),
            "kv_max": hi}


def _lengths(case):
    """(query tokens, key tokens) of each request: spread over the case's ranges, the last longest."""
    b = case["batch"]
    at = [(((i + 1) * 0.6180339887) % 1.0) if i + 1 < b else 1.0 for i in range(b)]
    q = [case["q_min"] + int(t * (case["q_max"] - case["q_min"])) for t in at]
    kv = [case["kv_min"] + int(t * (case["kv_max"] - case["kv_min"])) for t in at]
    return q, [n - (n == 3072) for n in kv]


# ---- inputs -------------------------------------------------------------------------------


def _tile_bytes(dim):
    return TILE * dim + 2 * TILE * (dim // GROUP) * 2


def _code_bytes(shape, gen):
    """Random cache codes, two in a byte: each 1..15, most near the middle, as values quantised by
    their group's largest are."""
    a = torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.uint8)
    b = torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.uint8)
    return (a & 0x77) + (b & 0x77) + 0x11


def _scales(shape, gen, size):
    """Random group scales of 8 significant bits and either sign, in f16."""
    d = torch.exp(0.3 * torch.randn(shape, generator=gen, device=DEV)) * size
    d = torch.where(torch.rand(shape, generator=gen, device=DEV) < 0.5, -d, d)
    return d.to(torch.bfloat16).to(torch.float16)


def _batch(case, gen):
    q, kv = _lengths(case)
    page = case["page"]
    per = max(1, -(-max(kv) // page))  # the widest request's pages
    b = case["batch"]
    perm = torch.randperm(b * per + 3, generator=gen, device=DEV)[: b * per]
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    tok_req = [i for i, n in enumerate(q) for _ in range(n)]
    tok_at = [j for n in q for j in range(n)]
    return {
        "q_len": q, "kv_len": kv, "max_q": max(q), "tokens": cu[-1], "n_pages": b * per + 3,
        "cu": torch.tensor(cu, dtype=torch.int32, device=DEV),
        "lens": torch.tensor(kv, dtype=torch.int32, device=DEV),
        "table": perm.to(torch.int32).reshape(b, per).contiguous(),
        # the plain forms index with these
        "req": torch.tensor(tok_req, dtype=torch.int64, device=DEV),
        "at": torch.tensor(tok_at, dtype=torch.int64, device=DEV),
    }


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    op = case["op"]
    s = {"case": case}
    if op == "norm":
        k, n = case["tokens"], case["n"]
        s["x"] = randn(k, n) * torch.exp(0.5 * randn(k, 1))
        s["x"][:, :: max(1, n // 7)] *= 12.0  # a residual stream has a few large channels
        s["add"] = randn(k, n) * 0.3 if case["add"] else None
        s["w"] = 1.0 + 0.2 * randn(n)
        s["resid"] = torch.empty(k, n, device=DEV)
        s["act"] = torch.empty(k, n, device=DEV, dtype=torch.bfloat16)
    elif op == "rope":
        s["b"] = b = _batch(case, gen)
        t, d = b["tokens"], case["dim"]
        s["q"] = randn(t, case["heads"], d)
        s["k"] = randn(t, case["kv_heads"], d) * torch.exp(0.7 * randn(case["kv_heads"], d))
        s["v"] = randn(t, case["kv_heads"], d)
        half = case["rot"] // 2
        angle = (torch.arange(max(b["kv_len"]) + 1, device=DEV, dtype=torch.float64)[:, None]
                 * 1e6 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half))
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).contiguous()
        rec = case["page"] // TILE * _tile_bytes(d)
        s["pages"] = torch.zeros(b["n_pages"], case["kv_heads"], rec, device=DEV,
                                 dtype=torch.uint8)
        s["q_out"] = torch.empty(t, case["heads"], d, device=DEV, dtype=TYPES[case["type"]])
        s["k_out"] = torch.empty(t, case["kv_heads"], d, device=DEV, dtype=torch.float16)
        s["v_out"] = torch.empty(t, case["kv_heads"], d, device=DEV, dtype=torch.float16)
    elif op == "attn":
        s["b"] = b = _batch(case, gen)
        d, tpp = case["dim"], case["page"] // TILE
        tiles = (b["n_pages"], case["kv_heads"], tpp)
        codes = _code_bytes((*tiles, TILE * d), gen)
        ks = _scales((*tiles, d // GROUP, TILE), gen, 0.45)
        vs = _scales((*tiles, d // GROUP, TILE), gen, 0.25)
        scales = torch.cat([ks.flatten(3), vs.flatten(3)], 3).contiguous().view(torch.uint8)
        s["pages"] = torch.cat([codes, scales], 3).reshape(b["n_pages"], case["kv_heads"], -1)
        s["pages"] = s["pages"].contiguous()
        s["q"] = randn(b["tokens"], case["heads"], d).to(TYPES[case["type"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = d ** -0.5
    else:
        r, v = case["rows"], case["vocab"]
        # a head's logits: a broad bulk and a few hundred likely tokens
        s["logits"] = randn(r, v) * 2.0
        likely = torch.randint(0, v, (r, 300), generator=gen, device=DEV)
        s["logits"].scatter_add_(1, likely, 3.0 * torch.rand(r, 300, generator=gen, device=DEV) + 4)
        s["u"] = torch.rand(r, generator=gen, device=DEV)
        s["t"] = 0.5 + torch.rand(r, generator=gen, device=DEV)
        s["top_k"] = torch.full((r,), case["top_k"], dtype=torch.int32, device=DEV)
        s["top_p"] = torch.full((r,), case["top_p"], device=DEV)
        s["min_p"] = torch.full((r,), case["min_p"], device=DEV)
        s["token"] = torch.empty(r, dtype=torch.int32, device=DEV)
        s["prob"] = torch.empty(r, device=DEV)
        s["kept"] = torch.empty(r, dtype=torch.int32, device=DEV)
    if own:  # the handles that a serving program keeps: the backend, the cache and the batch
        from apeiron_b200.step import DeviceAct, KV4Cache, SeqBatch

        s["ops"] = _step_ops()
        if op == "norm":
            s["codes"] = DeviceAct.empty(s["ops"], case["tokens"], case["n"])
        if "pages" in s:
            s["cache"] = KV4Cache(s["pages"], case["kv_heads"], case["dim"], case["page"])
            b = s["b"]
            s["batch"] = SeqBatch(b["cu"], b["lens"], b["table"], b["tokens"], b["max_q"])
    return s


_ops = None


def _step_ops():
    global _ops
    if _ops is None:
        from apeiron_b200 import Backend
        from apeiron_b200.step import StepOps

        _ops = StepOps(Backend(0))
    return _ops


# ---- one pass -----------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "rope": _own_rope, "attn": _own_attn,
                "sample": _own_sample}[op](s)
    return {"norm": _plain_norm, "rope": _plain_rope, "attn": _plain_attn,
            "sample": _plain_sample}[op](s)


def _own_norm(s):
    s["ops"].add_rms_norm_quant(s["x"], s["w"], 1e-6, add=s["add"], resid=s["resid"],
                                act=s["codes"], deq=s["act"])
    return {"act": s["act"], "resid": s["resid"]} if s["add"] is not None else {"act": s["act"]}


def _own_rope(s):
    c = s["case"]
    s["ops"].rope_kv4_append(s["q"], s["k"], s["v"], s["table"], s["cache"], s["batch"],
                             rot_dim=c["rot"], layout=c["layout"], q_out=s["q_out"],
                             k_deq=s["k_out"], v_deq=s["v_out"])
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "pages": s["pages"]}


def _own_attn(s):
    c = s["case"]
    s["ops"].attn_kv4(s["q"], s["cache"], s["batch"], s["scale"], window=c["window"],
                      sinks=c["sinks"], out=s["out"])
    return s["out"]


def _own_sample(s):
    s["ops"].sample(s["logits"], s["u"], temperature=s["t"], top_k=s["top_k"], top_p=s["top_p"],
                    min_p=s["min_p"], token=s["token"], prob=s["prob"], kept=s["kept"])
    return {"token": s["token"], "prob": s["prob"], "kept": s["kept"]}


# ---- plain forms --------------------------------------------------------------------------


def _blocks(y):
    """y's rows in groups of 32 lanes, zeros past the end."""
    k, n = y.shape
    return torch.nn.functional.pad(y, (0, -n % GROUP)).reshape(k, -1, GROUP)


def _plain_norm(s):
    x = s["x"] if s["add"] is None else s["x"] + s["add"]
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
    y = _blocks(x * r * s["w"])
    # S = 2^e / 2^32 with the smallest e >= 0 for which 127 S >= the group's largest
    big = torch.round(y.abs().amax(2, keepdim=True) * 2.0 ** 32)
    mant, e = torch.frexp(big)
    e = torch.clamp(e - 7 + (mant > 127.0 / 128.0).to(e.dtype), min=0)
    size = torch.ldexp(torch.full_like(big, 2.0 ** -32), e)
    code = torch.floor(y.abs() / size + 0.5)
    act = (torch.sign(y) * code * size).flatten(1)[:, : s["x"].shape[1]]
    act = act.to(torch.bfloat16)
    return {"act": act, "resid": x} if s["add"] is not None else {"act": act}


def _rotate(x, cs, rot, layout):
    """x (tokens, heads, dim) turned by cs (tokens, rot / 2, 2)."""
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    if layout == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _quantise4(x):
    """Codes and scales of x (..., dim): d = -m/8 for the group's largest value m, in 8 bits."""
    g = x.unflatten(-1, (-1, GROUP))
    hi, lo = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    d = (torch.where(hi >= -lo, hi, lo) * -0.125).to(torch.bfloat16).to(torch.float16)
    f = d.float()
    inv = torch.where(f == 0, f, 1.0 / f)
    return torch.clamp(torch.round(g * inv) + 8, 0, 15), d


def _plain_rope(s):
    c, b = s["case"], s["b"]
    dim, heads = c["dim"], c["kv_heads"]
    pos = (b["lens"].long() - (b["cu"][1:] - b["cu"][:-1]).long())[b["req"]] + b["at"]
    cs = s["table"][pos]
    q = _rotate(s["q"], cs, c["rot"], c["layout"]).to(TYPES[c["type"]])
    kc, kd = _quantise4(_rotate(s["k"], cs, c["rot"], c["layout"]))
    vc, vd = _quantise4(s["v"])
    k = ((kc - 8) * kd.float()).flatten(-2).to(torch.float16)
    v = ((vc - 8) * vd.float()).flatten(-2).to(torch.float16)
    # where each token's bytes go: page, then head, then tile, then its place in the tile
    page = b["table"][b["req"], pos // c["page"]].long()
    rec, tile = s["pages"].shape[2], _tile_bytes(dim)
    at = (page[:, None] * heads + torch.arange(heads, device=DEV)) * rec
    at = at + (pos % c["page"] // TILE * tile)[:, None]
    r = (pos % TILE)[:, None, None]
    kc, vc = kc.flatten(-2).to(torch.uint8), vc.flatten(-2).to(torch.uint8)
    i = torch.arange(dim // 2, device=DEV)
    k_at = at[..., None] + r * (dim // 2) + i
    k_byte = kc[..., 0::2] | kc[..., 1::2] << 4
    m, g = i // 8, i % 8  # this byte's 16-dim tile and its dim 16 m + g (and 16 m + g + 8)
    word = ((m // 4) * 32 + g * 4 + r % 8 // 2) * 4 + m % 4
    v_at = at[..., None] + TILE * dim // 2 + word * 4 + r % 2 * 2 + r // 8
    lanes = vc.unflatten(-1, (-1, 2, 8))
    v_byte = (lanes[..., 0, :] | lanes[..., 1, :] << 4).flatten(-2)
    j = torch.arange(2 * (dim // GROUP), device=DEV)
    s_at = at[..., None] + TILE * dim + (j // 2 * TILE + r) * 2 + j % 2
    flat = s["pages"].view(-1)
    flat[k_at] = k_byte
    flat[v_at] = v_byte
    flat[s_at] = kd.squeeze(-1).contiguous().view(torch.uint8)
    flat[s_at + TILE * (dim // GROUP) * 2] = vd.squeeze(-1).contiguous().view(torch.uint8)
    return {"q": q, "k": k, "v": v, "pages": s["pages"]}


def _gather_kv(s, dtype):
    """K and V of every request as (batch, kv heads, tokens, dim), from the pages of its table."""
    c, b = s["case"], s["b"]
    dim, heads, tpp = c["dim"], c["kv_heads"], c["page"] // TILE
    p = s["pages"][b["table"].long()].unflatten(-1, (tpp, -1))  # batch, page, head, tile, bytes
    p = p.transpose(1, 2).flatten(2, 3)                          # batch, head, tile, bytes
    n, half, sc = p.shape[2], TILE * dim // 2, TILE * (dim // GROUP)
    scales = p[..., 2 * half:].contiguous().view(torch.float16).to(dtype)
    ks = scales[..., :sc].unflatten(-1, (dim // GROUP, TILE)).transpose(-1, -2)
    vs = scales[..., sc:].unflatten(-1, (dim // GROUP, TILE)).transpose(-1, -2)
    kb = p[..., :half].unflatten(-1, (TILE, dim // 2))
    k = torch.stack([kb & 15, kb >> 4], -1).flatten(-2)          # batch, head, tile, token, dim
    vb = p[..., half: 2 * half].unflatten(-1, (dim // 64, 8, 4, 4, 2, 2))
    # (m / 4, g, t, m % 4, byte / 2, byte % 2) -> token = byte % 2 * 8 + t * 2 + byte / 2
    vb = torch.stack([vb & 15, vb >> 4], -1)                     # ..., dim + 8
    vb = vb.permute(0, 1, 2, 8, 5, 7, 3, 6, 9, 4)                # tokens, then m / 4, m % 4, +8, g
    v = vb.reshape(*p.shape[:2], n, TILE, dim)

    def values(code, scale):
        x = (code.to(dtype) - 8).unflatten(-1, (dim // GROUP, GROUP)) * scale[..., None]
        return x.flatten(-2).flatten(2, 3)

    return values(k, ks), values(v, vs)


def _plain_attn(s):
    c, b = s["case"], s["b"]
    q = s["q"]
    heads, groups, dim = c["heads"], c["heads"] // c["kv_heads"], c["dim"]
    k, v = _gather_kv(s, torch.float32)
    keys = k.shape[2]
    i = torch.arange(b["max_q"], device=DEV)
    n = (b["cu"][1:] - b["cu"][:-1]).long()
    rows = (b["cu"][:-1].long()[:, None] + i).clamp(max=q.shape[0] - 1)
    x = q.float()[rows].reshape(c["batch"], b["max_q"], c["kv_heads"], groups, dim)
    x = x.permute(0, 2, 3, 1, 4).reshape(c["batch"], c["kv_heads"], groups * b["max_q"], dim)
    p = (x @ k.transpose(-1, -2)) * s["scale"]
    p = p.reshape(c["batch"], c["kv_heads"], groups, b["max_q"], keys)
    pos = (b["lens"].long() - n)[:, None] + i
    j = torch.arange(keys, device=DEV)
    seen = j <= pos[..., None]
    if c["window"]:
        seen = seen & ((j < c["sinks"]) | (j > pos[..., None] - c["window"]))
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p.reshape(c["batch"], c["kv_heads"], groups * b["max_q"], keys)
    o = (p @ v).reshape(c["batch"], c["kv_heads"], groups, b["max_q"], dim)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(c["batch"], b["max_q"], heads, dim)
    return o[b["req"], b["at"]].to(q.dtype)


def _bits(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV).to(torch.int32).view(torch.float32)


def _exp32(x):
    """The framework's binary32 exp, one rounding for each operation."""
    n = torch.round(x * _bits(0x3fb8aa3b))
    r = x - n * _bits(0x3f318000) - n * _bits(0xb95e8083 - (1 << 32))
    p = _bits(0x39506967) * r + _bits(0x3ab743ce)
    p = p * r + _bits(0x3c088908)
    p = p * r + _bits(0x3d2aa9c1)
    p = p * r + _bits(0x3e2aaaaa)
    p = p * r + _bits(0x3f000000)
    y = (1.0 + r) + (r * r) * p
    n = n.clamp(-140, 140).to(torch.int32)
    a = n >> 1
    y = y * ((a + 127) << 23).view(torch.float32) * ((n - a + 127) << 23).view(torch.float32)
    return torch.where(x < -88.0, torch.zeros_like(y), y)


def _plain_sample(s):
    x = s["logits"]
    v = x.shape[1]
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(1, keepdim=True)
    z = torch.where(x == top, torch.zeros_like(x), x - top)
    e = _exp32(z * (1.0 / s["t"])[:, None])
    e = torch.where(x == -math.inf, torch.zeros_like(e), e)
    e, order = torch.sort(e, dim=1, descending=True, stable=True)
    w = torch.round(e * WEIGHT_ONE).long()
    rank = torch.arange(v, device=DEV)
    most = torch.where(s["top_k"] <= 0, torch.full_like(s["top_k"], v), s["top_k"])
    keep = rank < most[:, None]
    w = torch.where(keep, w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    limit = s["top_p"].double() * w.sum(1).double()
    cut = (s["top_p"] < 1)[:, None] & (before.double() >= limit[:, None]) & (rank > 0)
    keep = keep & ~cut
    keep = keep & (w.double() >= (s["min_p"].double() * WEIGHT_ONE)[:, None]) & (w > 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)  # back in the vocabulary's order
    run = torch.cumsum(w, 1)
    total = run[:, -1]
    aim = torch.minimum((s["u"].double() * total.double()).long(), total - 1)
    token = (run <= aim[:, None]).sum(1)
    prob = w.gather(1, token[:, None])[:, 0].double() / total.double()
    return {"token": token.int(), "prob": prob.float(), "kept": keep.sum(1).int()}


# ---- the definitions in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "attn": _exact_attn,
            "sample": _exact_sample}[case["op"]](s)


def _exact_norm(s):
    # the residual is a stored 32-bit value: the norm is of what is stored
    h = s["x"] if s["add"] is None else s["x"] + s["add"]
    x = h.double()
    y = x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / x.shape[1] + 1e-6) * s["w"].double()
    g = _blocks(y)
    fixed = torch.round(g * 4294967296.0)
    big = fixed.abs().amax(2, keepdim=True)
    e = torch.arange(63, device=DEV, dtype=torch.float64)
    e = (127.0 * 2.0 ** e < big).sum(2, keepdim=True)  # the smallest e with 127 2^e >= big
    size = 2.0 ** e.double()
    code = torch.sign(fixed) * torch.floor((2 * fixed.abs() + size) / (2 * size))
    act = (code * size / 4294967296.0).flatten(1)[:, : x.shape[1]]
    exact_sum = s["x"].double() if s["add"] is None else s["x"].double() + s["add"].double()
    return {"act": act, "resid": exact_sum} if s["add"] is not None else {"act": act}


def _exact_rope(s):
    c, b = s["case"], s["b"]
    first = [kv - q for q, kv in zip(b["q_len"], b["kv_len"])]
    pos = torch.tensor([f + j for f, q in zip(first, b["q_len"]) for j in range(q)], device=DEV)
    cs = s["table"].double()[pos]
    z = torch.complex(cs[..., 0], cs[..., 1])[:, None]

    def turn(x):
        x, rot = x.double().clone(), c["rot"]
        lanes = torch.arange(rot, device=DEV)
        a, o = (lanes[: rot // 2], lanes[rot // 2:]) if c["layout"] == "half" else (lanes[::2], lanes[1::2])
        y = torch.complex(x[..., a], x[..., o]) * z
        x[..., a], x[..., o] = y.real, y.imag
        return x

    def four(x):
        g = x.reshape(*x.shape[:-1], -1, 32)
        at = g.abs().argmax(-1, keepdim=True)
        m = g.gather(-1, at)
        d = (-m / 8).to(torch.bfloat16).to(torch.float16).double()
        code = torch.where(d == 0, torch.zeros_like(g), torch.round(g / torch.where(d == 0, torch.ones_like(d), d)))
        return (code.clamp(-8, 7) * d).reshape(x.shape)

    return {"q": turn(s["q"]), "k": four(turn(s["k"])), "v": four(s["v"]), "pages": None}


def _exact_attn(s):
    c, b = s["case"], s["b"]
    k, v = _gather_kv(s, torch.float64) if c["kv_max"] * c["batch"] * c["kv_heads"] < 400_000 else (None, None)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group, at = c["heads"] // c["kv_heads"], 0
    for i, (nq, nk) in enumerate(zip(b["q_len"], b["kv_len"])):
        if k is None:  # one request's pages at a time
            one = {**s, "b": {**b, "table": b["table"][i: i + 1]}}
            ki, vi = (t[0] for t in _gather_kv(one, torch.float64))
        else:
            ki, vi = k[i], v[i]
        pos = nk - nq + torch.arange(nq, device=DEV)
        j = torch.arange(nk, device=DEV)
        see = j[None] <= pos[:, None]
        if c["window"]:
            see &= (j[None] < c["sinks"]) | (j[None] > pos[:, None] - c["window"])
        for h in range(c["heads"]):
            if nk == 0:
                continue
            x = s["q"][at: at + nq, h].double() @ ki[h // group, :nk].T * s["scale"]
            x = torch.softmax(x.masked_fill(~see, -math.inf), -1)
            out[at: at + nq, h] = torch.nan_to_num(x, nan=0.0) @ vi[h // group, :nk]
        at += nq
    return out


def _exact_sample(s):
    prob = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        e = torch.exp((x - x.max()) / s["t"][r].double())
        w = torch.round(e * 2147483648.0)
        order = torch.argsort(e, descending=True, stable=True)
        k = s["case"]["top_k"] or x.numel()
        p, q = w[order[:k]], order[:k]
        limit = float(s["top_p"][r]) * float(p.sum()) if s["case"]["top_p"] < 1 else math.inf
        held = (p.cumsum(0) - p < limit) & (p >= float(s["min_p"][r]) * 2147483648.0)
        held[0] = True
        left = torch.zeros_like(w)
        left[q[held]] = p[held]
        run = left.cumsum(0)
        aim = math.floor(float(s["u"][r]) * float(run[-1]))
        prob.append(left[int((run <= aim).sum())] / run[-1])
    return {"token": None, "prob": torch.stack(prob), "kept": None}


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "norm":
        k, n = case["tokens"], case["n"]
        # x, (the addend, the new residual), weights, codes and scales, the dequantised values
        return {"bytes": k * n * (4 + (8 if case["add"] else 0) + 1 + 1 / 32 + 2) + 4 * n,
                "flops": 6 * k * n}
    if op == "sample":
        return {"bytes": 4 * case["rows"] * case["vocab"], "flops": 20 * case["rows"] * case["vocab"]}
    q, kv = _lengths(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["type"] == "f32" else 2
    if op == "rope":
        t = sum(q)
        return {"bytes": t * (h * d * (4 + size) + 2 * g * d * (4 + 0.5625 + 2) + case["rot"] * 4),
                "flops": t * d * (3 * h + 8 * g)}
    w, pairs, keys = case["window"], 0, 0
    for n, m in zip(q, kv):
        pos = range(m - n, m)
        if not w:
            pairs += sum(p + 1 for p in pos if p >= 0)
            keys += m
        else:
            pairs += sum(min(p + 1, w + min(case["sinks"], max(0, p + 1 - w))) for p in pos if p >= 0)
            first = max(0, m - n - w + 1)
            keys += m - first + min(case["sinks"], first)
    return {"bytes": keys * g * d * 2 * 0.5625 + 2 * sum(q) * h * d * size,
            "flops": 4 * d * h * pairs}
