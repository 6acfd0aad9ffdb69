"""The steps between the projections, written out plainly on the CPU (numpy, 64 bits and whole
numbers) from include/apeiron_cuda.h: what the GPU tests compare with."""
import math

import numpy as np

GROUP = 32
TILE = 16


# ---- the 4-bit cache, byte by byte ---------------------------------------------------------

def tile_bytes(dim):
    return TILE * dim + 2 * TILE * (dim // GROUP) * 2


def v_byte(i, r):
    m, g, t = i // 16, i % 8, (r % 8) // 2
    word = ((m // 4) * 32 + g * 4 + t) * 4 + m % 4
    return 4 * word + [2 * t, 2 * t + 8, 2 * t + 1, 2 * t + 9].index(r)


def read_token(pages, table_row, j, h, dim, page_tokens):
    """(k, v) of cached token j, KV head h: f64 vectors of d (c - 8)."""
    page = pages[table_row[j // page_tokens], h]
    r = j % page_tokens % TILE
    at = j % page_tokens // TILE * tile_bytes(dim)
    t = page[at: at + tile_bytes(dim)]
    scales = t[TILE * dim:].view(np.float16).astype(np.float64).reshape(2, dim // GROUP, TILE)
    k, v = np.empty(dim), np.empty(dim)
    for i in range(dim):
        b = int(t[r * (dim // 2) + i // 2])
        k[i] = ((b >> 4 if i % 2 else b & 15) - 8) * scales[0, i // GROUP, r]
        b = int(t[TILE * dim // 2 + v_byte(i, r)])
        v[i] = ((b >> 4 if i % 16 >= 8 else b & 15) - 8) * scales[1, i // GROUP, r]
    return k, v


def read_all(pages, table_row, n, h, dim, page_tokens):
    """K and V of tokens 0 .. n - 1, (n, dim) f64 each, by whole pages (read_token's values)."""
    if n == 0:
        return np.zeros((0, dim)), np.zeros((0, dim))
    used = pages[table_row[: -(-n // page_tokens)], h].reshape(-1, tile_bytes(dim))
    half = TILE * dim // 2
    kb = used[:, :half].reshape(-1, TILE, dim // 2)
    k = np.stack([kb & 15, kb >> 4], -1).reshape(-1, TILE, dim).astype(np.float64) - 8
    at = np.array([[v_byte(i, r) for i in range(dim)] for r in range(TILE)])
    vb = used[:, half: 2 * half][:, at]
    v = np.where(np.arange(dim) % 16 >= 8, vb >> 4, vb & 15).astype(np.float64) - 8
    sc = np.ascontiguousarray(used[:, 2 * half:]).view(np.float16).astype(np.float64)
    sc = sc.reshape(-1, 2, dim // GROUP, TILE).transpose(1, 0, 3, 2).repeat(GROUP, -1)
    return ((k * sc[0]).reshape(-1, dim)[:n], (v * sc[1]).reshape(-1, dim)[:n])


def attention(q, pages, table, q_lens, kv_lens, page_tokens, scale, window=0, sinks=0):
    """(out, reach, spread) in f64: the outputs (tokens, heads, dim), sum_j p_j |v_j| and, per
    (token, head), the largest scale * sum |q_d k_d| over the visible keys."""
    heads, dim = q.shape[1:]
    kv_heads = pages.shape[1]
    out = np.zeros(q.shape)
    reach, spread = np.zeros(q.shape), np.zeros(q.shape[:2])
    at = 0
    for s, (nq, nk) in enumerate(zip(q_lens, kv_lens)):
        kvs = [read_all(pages, table[s], nk, h, dim, page_tokens) for h in range(kv_heads)]
        for i in range(nq):
            pos = nk - nq + i
            j = np.arange(max(0, pos + 1))
            if window:
                j = j[(j < sinks) | (j > pos - window)]
            if j.size:
                for h in range(heads):
                    k, v = kvs[h // (heads // kv_heads)]
                    x = (k[j] @ q[at, h]) * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[at, h] = p @ v[j]
                    reach[at, h] = p @ np.abs(v[j])
                    spread[at, h] = abs(scale) * (np.abs(k[j]) @ np.abs(q[at, h])).max()
            at += 1
    return out, reach, spread


# ---- positions and the append ---------------------------------------------------------------

def rotate(x, cs, rot, layout):
    """x (heads, dim) f32 turned by cs (rot / 2, 2) f32, one rounding per operation."""
    x = x.astype(np.float32).copy()
    lanes = np.arange(rot)
    a, b = (lanes[: rot // 2], lanes[rot // 2:]) if layout == "half" else (lanes[::2], lanes[1::2])
    c, s = cs[:, 0], cs[:, 1]
    xa, xb = x[:, a].copy(), x[:, b].copy()
    x[:, a], x[:, b] = xa * c - xb * s, xb * c + xa * s
    return x


def to_bf16(x):
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + (u >> 16 & 1)) >> 16 << 16
    return u.astype(np.uint32).view(np.float32)


def four_bits(x):
    """The values d (c - 8) that x (..., dim) f32 is stored as."""
    g = x.reshape(*x.shape[:-1], -1, GROUP).astype(np.float32)
    hi, lo = g.max(-1, keepdims=True), g.min(-1, keepdims=True)
    m = np.where(hi >= -lo, hi, lo)
    d = to_bf16(m * np.float32(-0.125)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d)
    c = np.clip(np.rint(g * inv) + 8, 0, 15)
    return ((c - 8) * d).reshape(x.shape)


def frequencies(rot, base, scaling=None, factor=1.0, low=1.0, high=4.0, original=0.0):
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "bands":
            turns = original * f / (2 * math.pi)
            if turns < low:
                f /= factor
            elif turns <= high:
                s = (turns - low) / (high - low)
                f = f * (s + (1 - s) / factor)
        elif scaling == "ramp":
            def at(turns):
                return rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
            first, last = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
            s = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
            f = f * (1 - s) + f / factor * s
        out.append(f)
    return np.array(out)


# ---- the sampler, in whole numbers -----------------------------------------------------------

def exp32(x):
    """The F32 carrier's binary32 exp of a float32 vector."""
    f = lambda bits: np.uint32(bits).view(np.float32)  # noqa: E731
    x = np.asarray(x, np.float32)
    n = np.rint(x * f(0x3FB8AA3B))
    r = (x - n * f(0x3F318000)) - n * f(0xB95E8083)
    p = f(0x39506967) * r + f(0x3AB743CE)
    for c in (0x3C088908, 0x3D2AA9C1, 0x3E2AAAAA, 0x3F000000):
        p = p * r + f(c)
    y = (np.float32(1) + r) + (r * r) * p
    n = np.clip(n, -140, 140).astype(np.int32)
    a = n >> 1
    y = y * ((a + 127) << 23).view(np.float32) * ((n - a + 127) << 23).view(np.float32)
    return np.where(x < -88.0, np.float32(0), y)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, prob, kept) of one row."""
    x = np.where(np.isnan(logits), np.float32(-np.inf), logits).astype(np.float32)
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, 0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0, 1
    inv = np.float32(1) / np.float32(temperature)
    with np.errstate(invalid="ignore", over="ignore"):
        e = exp32(np.where(x == top, np.float32(0), (x - np.float32(top)) * inv))
    e = np.where(x == -np.inf, np.float32(0), e)
    w = [int(v) for v in np.rint(e.astype(np.float64) * 2.0 ** 31)]
    order = np.argsort(-e, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        limit = float(np.float32(top_p)) * float(sum(w[i] for i in order))
        left, before = [], 0
        for n, i in enumerate(order):
            if n and float(before) >= limit:
                break
            left.append(i)
            before += w[i]
        order = left
    least = float(np.float32(min_p)) * 2.0 ** 31
    keep = sorted(int(i) for i in order if w[i] > 0 and float(w[i]) >= least)
    total = sum(w[i] for i in keep)
    if not total:
        return -1, 0.0, 0
    aim = min(int(float(np.float32(u)) * float(total)), total - 1)
    run = 0
    for i in keep:
        run += w[i]
        if run > aim:
            return i, float(np.float32(w[i] / total)), len(keep)
