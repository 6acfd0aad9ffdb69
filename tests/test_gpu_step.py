"""The steps between the projections on the GPU (apeiron_b200.step) against tests/step_ref.py:
64-bit or whole-number restatements of include/apeiron_cuda.h.

Tolerances follow from the arithmetic, before any run:
- the norm's f32 output is one rounding of a value carried to more bits: one unit in the last
  place; its codes are exactly those of the column quantizer on that output;
- the rotation rounds each operation once and the 4-bit values are whole-number codes times an
  8-bit scale: equal bit for bit;
- attention in f32: a score is a sum of products good to 2^-22 of sum |q_d k_d| (two f16 halves
  of q, 22 bits), which moves a probability by twice that, and probabilities carry 22 bits and
  the sums 2^-21: 2^-21 spread + 2^-20 of sum p |v|, and a probability below 2^-38 of the row's
  largest may round to zero; the 16-bit types add one rounding of each probability to 11 bits
  (2^-11, and 2^-25 per key below f16's normal range) and the output's own rounding (2^-11 or
  2^-8);
- the sampler works in whole numbers: equal.
"""
import numpy as np
import pytest

import step_ref as ref

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


# ---- norm ---------------------------------------------------------------------------------

def norm_ref(h, w, eps):
    h = h.astype(np.float64)
    return h / np.sqrt((h * h).sum(1, keepdims=True) / h.shape[1] + eps) * w


def quantised(ops, y):
    """codes, exps, descs of the column quantizer on y (k, n) f32."""
    import torch

    k, n = y.shape
    pad = ops.lib.apx_act_padded_len(n)
    codes = torch.zeros(k, pad, dtype=torch.int8, device="cuda")
    exps = torch.full((k, pad // 32), 0xFF, dtype=torch.uint8, device="cuda")
    descs = torch.zeros(k, 8, dtype=torch.int32, device="cuda")
    assert ops.lib.apx_quant_f32_cols_async(ops.ctx, y.data_ptr(), n, k, codes.data_ptr(),
                                            exps.data_ptr(), descs.data_ptr(),
                                            torch.cuda.current_stream().cuda_stream) == 0
    return codes, exps, descs


@pytest.mark.parametrize("n", [1, 31, 32, 33, 100, 896, 1537, 4097, 8192, 12001, 40000])
@pytest.mark.parametrize("k,extra,add,weight", [(1, 0, True, True), (3, 0, False, True),
                                                (5, 3, True, False), (130, 4, True, True)])
def test_norm(ops, n, k, extra, add, weight):
    import torch
    from apeiron_b200.step import DeviceAct

    rng = np.random.default_rng(n * 7 + k)
    x = rng.standard_normal((k, n)).astype(np.float32) * np.exp(rng.standard_normal((k, 1)))
    x = x.astype(np.float32)
    x[:, :: max(1, n // 5)] *= 20
    if k > 2:
        x[1] = 0
    a = rng.standard_normal((k, n)).astype(np.float32) if add else None
    if add and k > 2:
        a[1] = 0
    w = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32) if weight else None

    def strided(v):  # rows `extra` elements further apart than they need be
        t = torch.full((k, n + extra), 7.0, device="cuda")[:, :n]
        t.copy_(gpu(v))
        return t

    y = strided(np.zeros((k, n), np.float32))
    resid = strided(np.zeros((k, n), np.float32)) if add else None
    deq = torch.empty(k, n, dtype=torch.bfloat16, device="cuda")
    act = DeviceAct.empty(ops, k, n)
    act.codes.fill_(99)
    ops.add_rms_norm_quant(strided(x), None if w is None else gpu(w), 1e-5,
                           add=strided(a) if add else None, resid=resid, act=act, deq=deq, y=y)
    h = x + a if add else x
    if add:
        assert np.array_equal(resid.cpu().numpy(), h)
    want = norm_ref(h, np.ones(n) if w is None else w.astype(np.float64), 1e-5)
    got = y.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 1e-44)
    codes, exps, descs = quantised(ops, y.contiguous())
    assert torch.equal(act.codes, codes)
    nb = -(-n // 32)
    assert torch.equal(act.exps[:, :nb], exps[:, :nb])
    assert torch.equal(act.descs, descs)
    e = exps[:, :nb].cpu().numpy().astype(np.int64)
    s = np.where(e == 0xFF, 0.0, np.ldexp(1.0, e - 32)).repeat(32, 1)[:, :n]
    stands = codes[:, :n].cpu().numpy() * s
    assert np.array_equal(deq.float().cpu().numpy().astype(np.float64), stands)


@pytest.mark.parametrize("n", [31, 896, 1537, 4097, 8192, 16001])
@pytest.mark.parametrize("k,extra,add,weight", [(149, 0, True, True), (301, 2, False, True)])
def test_norm_many_rows(ops, n, k, extra, add, weight):
    """More rows than the GPU has SMs."""
    test_norm(ops, n, k, extra, add, weight)


@pytest.mark.parametrize("k", [5, 160])
@pytest.mark.parametrize("n", [900, 5000])
@pytest.mark.parametrize("x_size,w_size,eps", [
    (1e18, 1e25, 1e-5), (1e37, 10.0, 1e-5), (1.0, 1e38, 1e-5), (1e-30, 1e-12, 0.0),
    (1e-36, 1e20, 0.0), (1e-20, 1e-30, 1e-30), (1e-3, 1e-38, 1e-12)])
def test_norm_far_numbers(ops, n, k, x_size, w_size, eps):
    """h w past f32's ends where y is not, and y itself past the upper one; y is rounded once, but
    for h w under the normal numbers, which lose up to 2^-150 before r < 2^20 lifts them."""
    import torch

    rng = np.random.default_rng(n + k)
    x = (rng.uniform(0.5, 2, (k, n)) * rng.choice([-1, 1], (k, n)) * x_size).astype(np.float32)
    w = (rng.uniform(0.5, 2, n) * w_size).astype(np.float32)
    y = torch.empty(k, n, device="cuda")
    ops.add_rms_norm_quant(gpu(x), gpu(w), eps, y=y, act=None)
    eps = np.float64(np.float32(eps))
    want = norm_ref(x, w.astype(np.float64), eps)
    got = y.cpu().numpy().astype(np.float64)
    r = 1 / np.sqrt((x.astype(np.float64) ** 2).mean(1, keepdims=True) + eps)
    bound = 2.0 ** -23 * np.abs(want) + 2.0 ** -149 * np.where(r < 2.0 ** 20, np.maximum(r, 1), 1)
    over = np.abs(want) > 3.4028235e38
    assert np.all(np.abs(got - want)[~over] <= bound[~over])
    assert np.all(np.abs(got[over]) >= 3.4028234e38)


def test_norm_in_place_and_refusals(ops):
    """resid = x; a row with NaN or Inf refuses as the quantizer does, the others do not; -1 rows
    stay apart; a row of any size, denormals among them."""
    import torch

    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 900)).astype(np.float32)
    x[1, 5], x[3, 899], x[4] = np.nan, np.inf, x[4] * 1e-41
    a = rng.standard_normal((6, 900)).astype(np.float32) * np.float32(0.5)
    a[4] = 0
    dx = gpu(x)
    y = torch.empty_like(dx)
    w = gpu(np.full(900, 2.0, np.float32))
    act = ops.add_rms_norm_quant(dx, w, 1e-12, add=gpu(a), resid=dx, y=y, act=None)
    assert act is None
    with np.errstate(all="ignore"):
        assert np.array_equal(dx.cpu().numpy(), x + a, equal_nan=True)
    act = ops.add_rms_norm_quant(dx, w, 1e-12)
    status = act.descs[:, 0].cpu().numpy()
    assert status.tolist() == [0, 10, 0, 10, 0, 0]
    fine = [0, 2, 4, 5]
    want = norm_ref((x + a)[fine], 2.0, 1e-12)
    got = y.cpu().numpy().astype(np.float64)[fine]
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 1e-44)


# ---- positions and the append -----------------------------------------------------------------

@pytest.mark.parametrize("scaling,kw", [
    (None, {}), ("linear", dict(factor=4.0)),
    ("bands", dict(factor=8.0, low=1.0, high=4.0, original=8192.0)),
    ("ramp", dict(factor=16.0, low=1.0, high=32.0, original=4096.0))])
@pytest.mark.parametrize("rot,base", [(128, 1e6), (32, 1e4)])
def test_rope_table(ops, scaling, kw, rot, base):
    n = 70001
    got = ops.rope_table(n, rot, base, scaling=scaling, mscale=1.25, **kw).cpu().numpy()
    f = ref.frequencies(rot, base, scaling, **kw)
    pos = np.r_[0:40, 4095:4100, n - 20:n]
    a = pos[:, None] * f
    want = np.stack([np.cos(a), np.sin(a)], -1) * 1.25
    # one f32 rounding of a value below 1.25, and the f64 angle's (2^-52 of 7e4, twice)
    assert np.abs(got[pos] - want).max() <= 2.0 ** -24 * 1.25 + 7e4 * 2.0 ** -50


def batch_of(q_lens, kv_lens, page, rng, spare=2, wide=0):
    """(SeqBatch, table, n_pages): pages in random order."""
    from apeiron_b200.step import SeqBatch

    per = max(1, max(-(-n // page) for n in kv_lens)) + wide
    n = len(q_lens)
    perm = rng.permutation(n * per + spare)[: n * per].astype(np.int32).reshape(n, per)
    cu = np.r_[0, np.cumsum(q_lens)].astype(np.int32)
    b = SeqBatch(gpu(cu), gpu(np.array(kv_lens, np.int32)), gpu(perm), int(cu[-1]),
                 max(max(q_lens), 1))
    return b, perm, n * per + spare


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(14, 2, 64, 16), (12, 2, 128, 64),
                                                     (5, 5, 64, 128), (8, 1, 128, 32)])
@pytest.mark.parametrize("rot,layout,kind", [(64, "half", "float32"), (64, "interleaved", "float16"),
                                             (24, "half", "bfloat16"), (8, "interleaved", "bfloat16"),
                                             (0, "half", "float32")])
def test_rope_append(ops, heads, kv_heads, dim, page, rot, layout, kind):
    import torch
    from apeiron_b200.step import KV4Cache

    rng = np.random.default_rng(heads * 100 + rot)
    q_lens, kv_lens = [1, 0, 5, 37, 1], [1, 9, 70, 37, 200]
    b, table, n_pages = batch_of(q_lens, kv_lens, page, rng, wide=1)
    t = sum(q_lens)
    # q, k and v as slices of one fused row
    width = (heads + 2 * kv_heads) * dim
    fused = rng.standard_normal((t, width)).astype(np.float32) * np.float32(3)
    fused[2, heads * dim: heads * dim + 32] = 0            # a group of zeros
    fused[3, heads * dim: heads * dim + 32] = 1e-9         # one below every scale
    fused[4, -32:] = np.r_[5, -5, np.zeros(30)]            # two of the same magnitude
    dev = gpu(fused)
    q = dev[:, : heads * dim].unflatten(1, (heads, dim))
    k = dev[:, heads * dim: (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    v = dev[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
    tab = ops.rope_table(256, rot, 1e4) if rot else torch.empty(256, 0, 2, device="cuda")
    cache = KV4Cache.empty(n_pages, kv_heads, dim, page)
    cache.pages.fill_(0xA5)
    deq = [torch.empty(t, kv_heads, dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    status = ops.new_status()
    out = ops.rope_kv4_append(q, k, v, tab, cache, b, rot_dim=rot, layout=layout,
                              q_type=getattr(torch, kind), k_deq=deq[0], v_deq=deq[1],
                              status=status)
    assert ops.check_status(status) is None
    cs, pages = tab.cpu().numpy(), cache.pages.cpu().numpy()
    touched = np.zeros(pages.shape[:2] + (page,), bool)
    i = 0
    for s, (nq, nk) in enumerate(zip(q_lens, kv_lens)):
        for j in range(nk - nq, nk):
            qw = torch.from_numpy(ref.rotate(q[i].cpu().numpy(), cs[j], rot, layout))
            assert torch.equal(out[i].cpu(), qw.to(getattr(torch, kind)))
            kw = ref.four_bits(ref.rotate(k[i].cpu().numpy(), cs[j], rot, layout))
            vw = ref.four_bits(v[i].cpu().numpy())
            assert np.array_equal(deq[0][i].float().cpu().numpy(), kw)
            assert np.array_equal(deq[1][i].float().cpu().numpy(), vw)
            for h in range(kv_heads):
                got = ref.read_token(pages, table[s], j, h, dim, page)
                assert np.array_equal(got[0], kw[h]) and np.array_equal(got[1], vw[h])
                touched[table[s, j // page], h, j % page] = True
            i += 1
    # nothing else was written: every tile without a token still holds the fill
    tiles = pages.reshape(*pages.shape[:2], page // 16, -1)
    clean = ~touched.reshape(*touched.shape[:2], page // 16, 16).any(-1)
    assert (tiles[clean] == 0xA5).all()


def test_rope_append_refusals(ops):
    """Positions outside the table or the cache, pages outside it, values without a 4-bit image:
    the first token's refusal in the status, nothing written for it, the others served."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(1)
    cache = KV4Cache.empty(4, 1, 64, 16)
    tab = ops.rope_table(40, 64)
    k = gpu(rng.standard_normal((4, 1, 64)).astype(np.float32))

    def call(kv_len, table, k=k):
        cache.pages.fill_(0x11)
        status = ops.new_status()
        cu = gpu(np.arange(5, dtype=np.int32))
        b = SeqBatch(cu, gpu(np.array(kv_len, np.int32)), gpu(np.array(table, np.int32)), 4, 1)
        assert ops.rope_kv4_append(None, k, k, tab, cache, b, rot_dim=64, status=status) is None
        pages = cache.pages.cpu().numpy()
        return ops.check_status(status), [(pages[p] != 0x11).any() for p in range(4)]

    ok = [[0, 0, 0], [1, 1, 1], [2, 2, 2], [3, 3, 3]]
    assert call([1, 17, 40, 3], ok) == (None, [True] * 4)
    assert call([1, 41, 40, 3], ok) == ((1, 20), [True, False, True, True])   # past the table
    assert call([1, 17, 0, 3], ok) == ((2, 20), [True, True, False, True])    # before token 0
    assert call([1, 17, 40, 49], ok)[0] == (3, 20)                            # past its pages
    bad = [[0, 0, 0], [1, 4, 1], [2, 2, -1], [3, 3, 3]]
    assert call([1, 17, 40, 3], bad) == ((1, 20), [True, False, False, True])
    for value in (np.nan, np.inf, -70000.0):
        x = k.clone()
        x[2, 0, 33] = value
        got, wrote = call([1, 17, 40, 3], ok, x)
        assert got == (2, 10) and all(wrote)
        # the refused group stands for zeros, the other group and the other tokens as ever
        pages = cache.pages.cpu().numpy()
        kk, vv = ref.read_token(pages, [2, 2, 2], 39, 0, 64, 16)
        assert not vv[32:].any() and np.array_equal(vv[:32], ref.four_bits(x[2].cpu().numpy())[0, :32])


# ---- attention ----------------------------------------------------------------------------------

def random_pages(n_pages, kv_heads, dim, page, rng, k_size=0.4, v_size=0.3):
    tiles = (n_pages, kv_heads, page // 16)
    codes = rng.integers(0, 256, (*tiles, 16 * dim), dtype=np.uint8)
    d = np.exp(0.4 * rng.standard_normal((*tiles, 2, dim // 32, 16)))
    d *= np.array([k_size, v_size])[:, None, None] * rng.choice([-1, 1], d.shape)
    d = ref.to_bf16(d).astype(np.float16).reshape(*tiles, -1).view(np.uint8)
    return np.ascontiguousarray(np.concatenate([codes, d], -1).reshape(n_pages, kv_heads, -1))


def spoil(pages, table, kv_lens, dim, page):
    """Every token that no sequence holds: 0xFF bytes, whose scales are NaN."""
    held = np.zeros((pages.shape[0], page), bool)
    for s, n in enumerate(kv_lens):
        for j in range(n):
            held[table[s, j // page], j % page] = True
    p = pages.reshape(*pages.shape[:2], page // 16, ref.tile_bytes(dim))
    for r in range(page):
        free = ~held[:, r]
        at = p[:, :, r // 16]
        sc = np.array([16 * dim + (g * 16 + r % 16) * 2 + b
                       for g in range(2 * dim // 32) for b in range(2)])
        k = np.arange(r % 16 * dim // 2, (r % 16 + 1) * dim // 2)
        v = 8 * dim + np.array([ref.v_byte(i, r % 16) for i in range(0, dim)])
        for cols in (sc, k, v):
            at[np.ix_(free, range(at.shape[1]), cols)] = 0xFF


def check_attention(ops, q_lens, kv_lens, heads, kv_heads, dim, page, kind, window=0, sinks=0,
                    scale=None, seed=0, stream=None, k_size=0.4):
    import torch
    from apeiron_b200.step import KV4Cache

    rng = np.random.default_rng(seed + 17 * dim + heads)
    b, table, n_pages = batch_of(q_lens, kv_lens, page, rng)
    pages = random_pages(n_pages, kv_heads, dim, page, rng, k_size)
    spoil(pages, table, kv_lens, dim, page)
    t = sum(q_lens)
    dt = getattr(torch, kind)
    # q and out as slices of wider rows
    q = gpu(rng.standard_normal((t, heads + 2, dim)).astype(np.float32)).to(dt)[:, 1: heads + 1]
    out = torch.full((t, heads + 1, dim), 3.0, dtype=dt, device="cuda")[:, :heads]
    scale = dim ** -0.5 if scale is None else scale
    cache = KV4Cache(gpu(pages), kv_heads, dim, page)
    status = ops.new_status()
    torch.cuda.synchronize()
    ops.attn_kv4(q, cache, b, scale, window=window, sinks=sinks, out=out, status=status,
                 stream=stream)
    torch.cuda.synchronize()
    assert ops.check_status(status) is None
    again = torch.empty_like(q.contiguous())
    ops.attn_kv4(q, cache, b, scale, window=window, sinks=sinks, out=again)
    assert torch.equal(out, again)  # the same bits each time
    want, reach, spread = ref.attention(q.double().cpu().numpy(), pages, table, q_lens, kv_lens,
                                        page, scale, window, sinks)
    got = out.double().cpu().numpy()
    tol = (2.0 ** -21 * spread + 2.0 ** -20)[..., None] * reach
    tol = tol + 2.0 ** -38 * max(kv_lens) * pages_max(pages, dim)
    if kind != "float32":
        tol = tol + 2.0 ** -11 * reach + 2.0 ** -25 * max(kv_lens) * pages_max(pages, dim)
        tol = tol + (2.0 ** -11 if kind == "float16" else 2.0 ** -8) * np.abs(want)
        tol = tol + (2.0 ** -24 if kind == "float16" else 0)
    over = np.abs(got - want) - tol
    assert np.isfinite(got).all() and over.max() <= 0, (over.max(), np.abs(got - want).max())


def pages_max(pages, dim):
    sc = pages.reshape(-1, ref.tile_bytes(dim))[:, 16 * dim:].copy().view(np.float16)
    return 8 * float(np.nanmax(np.abs(sc.astype(np.float32))))


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (14, 2, 64, 16), (12, 2, 128, 64), (16, 2, 128, 32), (3, 3, 64, 128), (16, 1, 64, 64),
    (64, 8, 128, 16), (20, 1, 128, 16)])
def test_attention_decode(ops, kind, heads, kv_heads, dim, page):
    """Single tokens over contexts of every residue of a tile and a page, none at all included."""
    kv = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 255, 300]
    check_attention(ops, [1] * len(kv), kv, heads, kv_heads, dim, page, kind)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [1, 777, 5000, 33333])
def test_attention_long_context(ops, kind, n):
    """One request, its keys split over the GPU; one 100 times the other's length."""
    check_attention(ops, [1], [n], 8, 1, 128, 64, kind, seed=n)
    check_attention(ops, [1, 1], [n, n // 100], 14, 2, 64, 16, kind, seed=n + 1)


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(14, 2, 64, 16), (12, 2, 128, 64),
                                                     (4, 4, 64, 32), (16, 1, 128, 128)])
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([5], [5]), ([2, 3, 1, 0, 4], [40, 3, 17, 20, 150]), ([130], [130]), ([100, 17], [300, 17]),
    ([257, 64, 1], [400, 64, 511])])
def test_attention_prefill(ops, kind, heads, kv_heads, dim, page, q_lens, kv_lens):
    check_attention(ops, q_lens, kv_lens, heads, kv_heads, dim, page, kind)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(14, 2, 64, 16), (16, 1, 128, 128), (12, 2, 128, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1100, 0), (300, 5)])
@pytest.mark.parametrize("q_lens,kv_lens", [([14], [1025]), ([30], [4001]), ([100, 3, 20], [2500, 900, 20]),
                                            ([130], [1300])])
def test_attention_chunk_of_long(ops, kind, heads, kv_heads, dim, page, window, sinks, q_lens, kv_lens):
    """Few blocks of rows over long contexts, whose keys several CTAs share."""
    check_attention(ops, q_lens, kv_lens, heads, kv_heads, dim, page, kind, window, sinks)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 0), (100, 33), (5000, 4),
                                          (64, 64)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [300, 7, 1000]), ([90, 3], [400, 50]),
                                            ([260], [700])])
def test_attention_window(ops, kind, window, sinks, q_lens, kv_lens):
    check_attention(ops, q_lens, kv_lens, 14, 2, 64, 16, kind, window, sinks)
    check_attention(ops, q_lens, kv_lens, 8, 2, 128, 64, kind, window, sinks)


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("q_lens,kv_lens", [([3, 1], [1, 0]), ([200], [150])])
def test_attention_queries_before_the_first_key(ops, kind, q_lens, kv_lens):
    """More query tokens than cached ones: the first stand before token 0 and get zeros."""
    check_attention(ops, q_lens, kv_lens, 8, 2, 64, 16, kind)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale,k_size", [(3.0, 2.0), (0.0, 0.4), (-0.5, 0.4)])
def test_attention_scores_of_any_size(ops, kind, scale, k_size):
    """Scores in the hundreds (one key takes all), all equal, and of the other sign."""
    check_attention(ops, [1, 1], [100, 500], 8, 2, 64, 16, kind, scale=scale, k_size=k_size)
    check_attention(ops, [140], [300], 8, 2, 64, 16, kind, scale=scale, k_size=k_size)


def test_attention_on_another_stream(ops):
    import torch

    s = torch.cuda.Stream()
    check_attention(ops, [1, 1], [900, 80], 12, 2, 128, 64, "float32", stream=s.cuda_stream)
    check_attention(ops, [150], [190], 12, 2, 128, 64, "bfloat16", stream=s.cuda_stream)


@pytest.mark.parametrize("nq", [1, 150])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_attention_pages_outside_the_cache(ops, nq, kind):
    """A page number outside the cache is reported with its sequence, and not read."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(2)
    cache = KV4Cache(gpu(random_pages(8, 2, 64, 64, rng)), 2, 64, 64)
    q = torch.randn(2 * nq, 4, 64, device="cuda").to(getattr(torch, kind))
    for page in (-1, 8, 1 << 30):
        table = np.array([[0, 1, 2], [3, page, 5]], np.int32)
        b = SeqBatch(gpu(np.array([0, nq, 2 * nq], np.int32)),
                     gpu(np.array([180, 190], np.int32)), gpu(table), 2 * nq, nq)
        status = ops.new_status()
        ops.attn_kv4(q, cache, b, 0.1, status=status)
        assert ops.check_status(status) == (1, 20)
    # lengths past the table's pages
    b = SeqBatch(gpu(np.array([0, nq, 2 * nq], np.int32)), gpu(np.array([193, 190], np.int32)),
                 gpu(np.array([[0, 1, 2], [3, 4, 5]], np.int32)), 2 * nq, nq)
    status = ops.new_status()
    ops.attn_kv4(q, cache, b, 0.1, status=status)
    assert ops.check_status(status) == (0, 20)


# ---- the sampler ---------------------------------------------------------------------------------

def check_sample(ops, logits, u, pad=0, **kw):
    import torch

    rows, vocab = logits.shape
    x = torch.full((rows, vocab + pad), 9e9, device="cuda")[:, :vocab]
    x.copy_(gpu(logits))
    per = {k: np.broadcast_to(np.asarray(v, np.int32 if k == "top_k" else np.float32), (rows,))
           for k, v in kw.items()}
    prob = torch.empty(rows, device="cuda")
    kept = torch.empty(rows, dtype=torch.int32, device="cuda")
    u = np.broadcast_to(np.asarray(u, np.float32), (rows,))
    token = ops.sample(x, gpu(u), prob=prob, kept=kept, **{k: gpu(v) for k, v in per.items()})
    got = list(zip(token.tolist(), prob.tolist(), kept.tolist()))
    want = [ref.sample(logits[r], u[r], **{k: v[r] for k, v in per.items()}) for r in range(rows)]
    assert got == want


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_k=10 ** 9), dict(top_p=0.0),
           dict(top_p=0.3), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
           dict(top_k=40, top_p=0.9, min_p=0.01, temperature=0.7),
           dict(top_p=0.8, temperature=5.0), dict(top_k=3, top_p=1e-6, temperature=0.05)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 32003])
@pytest.mark.parametrize("f", FILTERS, ids=str)
def test_sample(ops, vocab, f):
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((6, vocab)) * 3).astype(np.float32)
    check_sample(ops, logits, [0.0, 0.1, 0.5, 0.9, 0.999, 1 - 2.0 ** -24], pad=vocab % 5, **f)


@pytest.mark.parametrize("vocab", [151936, 300001, 524288])
def test_sample_large_vocabulary(ops, vocab):
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((3, vocab)) * 2).astype(np.float32)
    logits[:, :: vocab // 50] += 8
    for f in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95, min_p=0.02),
              dict(top_k=100000, temperature=3.0)):
        check_sample(ops, logits, [0.2, 0.7, 0.97], **f)


@pytest.mark.parametrize("rows,vocab", [(90, 32003), (45, 65535), (24, 151936), (12, 300001)])
def test_sample_many_rows(ops, rows, vocab):
    """More CTAs than the GPU has SMs; flat rows, whose nuclei fit no list, among peaked ones."""
    rng = np.random.default_rng(rows)
    logits = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    logits[::2, :: vocab // 70] += 9
    u = (np.arange(rows) + 0.5) / rows
    for f in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.93, min_p=0.02),
              dict(top_k=3001, top_p=0.8)):
        check_sample(ops, logits, u, **f)


@pytest.mark.parametrize("f", FILTERS, ids=str)
def test_sample_ties(ops, f):
    """Few different logits: the lower index comes first of equals, at every cut."""
    rng = np.random.default_rng(8)
    logits = rng.integers(0, 4, (8, 5003)).astype(np.float32)
    logits[6] = 2.5          # all equal
    logits[7, 1:] = -30.0    # one token, and a level far below
    check_sample(ops, logits, np.linspace(0.001, 0.999, 8), **f)


@pytest.mark.parametrize("f", FILTERS, ids=str)
def test_sample_special_values(ops, f):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((9, 2000)).astype(np.float32)
    inf = np.float32(np.inf)
    x[0, ::3] = -inf
    x[1, ::2] = np.nan
    x[2] = -inf                       # nothing
    x[3] = np.nan                     # nothing
    x[4, [5, 900, 1999]] = inf        # only these
    x[5] = -3.4e38                    # the type's lowest value
    x[6, 100:] = -3.4e38
    x[7, 1:] = -inf                   # one
    x[8] = 3.4e38
    check_sample(ops, x, 0.6, **f)


@pytest.mark.parametrize("t", [0.0, -1.0, 1e-3, 1e-30, 1e30, np.inf, np.nan])
def test_sample_temperatures(ops, t):
    rng = np.random.default_rng(10)
    x = (rng.standard_normal((4, 3001)) * 4).astype(np.float32)
    x[2, 1000:] = x[2].max()
    check_sample(ops, x, [0.1, 0.4, 0.7, 0.99], temperature=t)
    check_sample(ops, x, [0.1, 0.4, 0.7, 0.99], temperature=t, top_k=20, top_p=0.7)


def test_sample_frequencies(ops):
    """20000 evenly spread numbers draw each of 8 tokens as often as its probability says."""
    import torch

    x = np.log(np.array([1, 2, 3, 4, 5, 6, 7, 8], np.float32)).astype(np.float32)
    n = 20000
    u = (np.arange(n) + 0.5) / n
    token = ops.sample(gpu(np.tile(x, (n, 1))), gpu(u.astype(np.float32)))
    count = torch.bincount(token.long(), minlength=8).cpu().numpy()
    assert np.abs(count - n * np.arange(1, 9) / 36).max() <= 1.5


# ---- refusals on the host ---------------------------------------------------------------------

def test_refusals(ops):
    import torch
    from apeiron_b200 import _abi
    from apeiron_b200.step import KV4Cache, SeqBatch

    x = torch.zeros(4, 64, device="cuda")
    w = torch.zeros(64, device="cuda")
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x.double(), w, 1e-6)
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x, w[:63], 1e-6)
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x.t(), torch.zeros(4, device="cuda"), 1e-6)  # rows not contiguous
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x, w, -1.0)
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x, w, 1e-6, deq=x.half())
    with pytest.raises(ValueError):
        KV4Cache.empty(4, 2, 80, 16)
    with pytest.raises(ValueError):
        KV4Cache.empty(4, 2, 64, 24)
    cache = KV4Cache.empty(4, 2, 64, 16)
    i32 = dict(dtype=torch.int32, device="cuda")
    b = SeqBatch(torch.tensor([0, 4], **i32), torch.tensor([4], **i32),
                 torch.zeros(1, 1, **i32), 4, 4)
    q = torch.zeros(4, 4, 64, device="cuda")
    k = torch.zeros(4, 2, 64, device="cuda")
    tab = ops.rope_table(16, 64)
    for kw in (dict(rot_dim=12), dict(rot_dim=72), dict(rot_dim=64, layout="other")):
        with pytest.raises(ValueError):
            ops.rope_kv4_append(q, k, k, tab, cache, b, **kw)
    with pytest.raises(ValueError):
        ops.rope_kv4_append(q, k[:, :1], k, tab, cache, b, rot_dim=64)
    with pytest.raises(ValueError):
        ops.attn_kv4(torch.zeros(4, 3, 64, device="cuda"), cache, b, 1.0)  # 3 heads on 2
    with pytest.raises(ValueError):
        ops.attn_kv4(q.double(), cache, b, 1.0)
    with pytest.raises(ValueError):
        ops.attn_kv4(q, cache, b, 1.0, window=-1)
    with pytest.raises(ValueError):
        ops.attn_kv4(q, cache, b, float("nan"))
    with pytest.raises(ValueError):  # rows that do not start on 16 bytes
        ops.attn_kv4(torch.zeros(4, 4 * 64 + 1, device="cuda")[:, 1:].unflatten(1, (4, 64)),
                     cache, b, 1.0)
    with pytest.raises(ValueError):
        ops.attn_kv4(q, cache, SeqBatch(b.cu, b.kv_len, b.table, 4, 5), 1.0)  # max_q > tokens
    with pytest.raises(ValueError):
        ops.rope_table(16, 7)
    with pytest.raises(ValueError):
        ops.rope_table(16, 64, scaling="bands", factor=2.0, low=4.0, high=1.0, original=1.0)
    u = torch.zeros(1, device="cuda")
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(1, _abi.SAMPLE_MAX_VOCAB + 1, device="cuda"), u)
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(2, 10, device="cuda"), u)
    # no rows: nothing to do
    assert ops.sample(torch.zeros(0, 10, device="cuda"), u[:0]).numel() == 0
    e = SeqBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 1, **i32), 0, 0)
    assert ops.attn_kv4(q[:0], cache, e, 1.0).numel() == 0
