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


# ---- lengths and bounds that do not fit ------------------------------------------------------

@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("q_lens,max_q", [([1, 3, 1], 2), ([8, 9, 1], 8), ([20, 41, 2], 40),
                                          ([256, 257, 9], 256), ([600, 700, 128], 128)])
def test_attention_more_queries_than_max_q(ops, kind, q_lens, max_q):
    """A sequence with more query tokens than the batch says is refused with its number; the others
    get what a batch whose bound fits gives them, to the roundings of another split."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(max_q)
    kv_lens = [n + 30 for n in q_lens]
    good, table, n_pages = batch_of(q_lens, kv_lens, 16, rng)
    cache = KV4Cache(gpu(random_pages(n_pages, 2, 64, 16, rng)), 2, 64, 16)
    q = torch.randn(sum(q_lens), 2, 64, device="cuda").to(getattr(torch, kind))
    stale = SeqBatch(good.cu, good.kv_len, good.table, good.n_tokens, max_q)
    status = ops.new_status()
    ops.attn_kv4(q, cache, stale, 0.1, status=status)
    first = [i for i, n in enumerate(q_lens) if n > max_q][0]
    assert ops.check_status(status) == (first, 20)
    status = ops.new_status()
    out = ops.attn_kv4(q, cache, stale, 0.1)
    want = ops.attn_kv4(q, cache, good, 0.1, status=status)
    assert ops.check_status(status) is None
    cu = np.r_[0, np.cumsum(q_lens)]
    for i, n in enumerate(q_lens):
        if n <= max_q:
            a, b = (t[cu[i]: cu[i + 1]].double() for t in (out, want))
            assert (a - b).abs().max() <= 2.0 ** -7 * b.abs().max()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("q_lens", [[70], [3, 1, 2], [1, 1, 1]])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_steps_numbered_in_64_bits(ops, kind, q_lens, window):
    """A table with room for more keys than 32 bits of steps: the call that numbers them in 64.  A
    prompt's blocks get the bits they get with a small table; single tokens, which then go in blocks
    of more rows, the same to f32's or the type's roundings."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(len(q_lens))
    n, heads = len(q_lens), 16
    kv_lens = [n_q + 300 + 17 * i for i, n_q in enumerate(q_lens)]
    small, table, n_pages = batch_of(q_lens, kv_lens, 128, rng)
    wide = torch.zeros(n, 25_000_000 if n > 1 else 60_000_000, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = gpu(table)
    batch = SeqBatch(small.cu, small.kv_len, wide, small.n_tokens, max(q_lens))
    blocks = n if max(q_lens) == 1 else sum(q_lens) // 16 + 2 * n
    assert blocks * heads * (wide.shape[1] * 128 // 32) >= 2 ** 32
    cache = KV4Cache(gpu(random_pages(n_pages, heads, 64, 128, rng)), heads, 64, 128)
    q = torch.randn(sum(q_lens), heads, 64, device="cuda").to(getattr(torch, kind))
    status = ops.new_status()
    got = ops.attn_kv4(q, cache, batch, 0.125, window=window, status=status)
    want = ops.attn_kv4(q, cache, small, 0.125, window=window)
    assert ops.check_status(status) is None
    if max(q_lens) > 8:
        assert torch.equal(got, want)
    else:
        off = (got.double() - want.double()).abs().max() / want.double().abs().max()
        assert off <= (2.0 ** -16 if kind == "float32" else 2.0 ** -7)


# ---- pages behind every window ---------------------------------------------------------------

@pytest.mark.parametrize("kind", ["float32", "float16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (64, 32), (128, 64), (64, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 0), (100, 5), (64, 20), (250, 16)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [300, 7, 1000]), ([9, 3], [400, 350]),
                                            ([60, 20], [500, 300]), ([260], [800])])
def test_attention_without_the_pages_behind_the_window(ops, kind, dim, page, window, sinks, q_lens,
                                                       kv_lens):
    """Pages of which no query sees a key are out of the table: numbers outside the cache, or a page
    whose scales are NaN.  The other values behind the windows are NaN too."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(window + dim)
    b, table, n_pages = batch_of(q_lens, kv_lens, page, rng)
    pages = random_pages(n_pages, 2, dim, page, rng)
    q = gpu(rng.standard_normal((sum(q_lens), 4, dim)).astype(np.float32)).to(getattr(torch, kind))
    want, reach, spread = ref.attention(q.double().cpu().numpy(), pages, table, q_lens, kv_lens,
                                        page, 0.2, window, sinks)
    left = table.copy()
    free = [p for p in range(n_pages) if p not in table]
    pages[free] = 0xFF
    tiles = pages.reshape(n_pages, 2, page // 16, -1)
    for s, (nq, nk) in enumerate(zip(q_lens, kv_lens)):
        low = nk - nq - window + 1
        for j in range(sinks, low):  # the scales of every unseen token
            at = 16 * dim + (np.arange(2 * dim // 32)[:, None] * 16 + j % 16) * 2 + np.arange(2)
            tiles[table[s, j // page], :, j % page // 16, at.ravel()] = 0xFF
        for i in range(table.shape[1]):
            if i * page >= sinks and (i + 1) * page <= low:
                left[s, i] = rng.choice([-1, n_pages, 1 << 30, free[0]])
    if max(q_lens) < 100:
        assert (left != table).any() or window == 250
    cache = KV4Cache(gpu(pages), 2, dim, page)
    status = ops.new_status()
    out = ops.attn_kv4(q, cache, SeqBatch(b.cu, b.kv_len, gpu(left), sum(q_lens), max(q_lens)), 0.2,
                       window=window, sinks=sinks, status=status)
    assert ops.check_status(status) is None
    got = out.double().cpu().numpy()
    # check_attention's bounds
    most = 8 * 0.3 * np.exp(0.4 * 6)
    tol = (2.0 ** -21 * spread + 2.0 ** -20)[..., None] * reach + 2.0 ** -38 * max(kv_lens) * most
    if kind != "float32":
        tol = tol + 2.0 ** -11 * reach + 2.0 ** -25 * max(kv_lens) * most
        tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -24
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


# ---- the append's lengths -------------------------------------------------------------------

@pytest.mark.parametrize("cu,kv_len,first", [
    ([0, 2, 4], [10, 20], 4),                     # two tokens behind the last request
    ([0, 0, 0], [10, 20], 0),                     # none of them in a request
    ([3, 4, 6], [10, 20], 0),                     # three before the first
    ([0, 2, 6], [10, -2 ** 31], 2), ([0, 2, 6], [-1, 20], 0), ([0, 2, 6], [10, 3], 2)])
def test_append_tokens_of_no_request(ops, cu, kv_len, first):
    """Tokens that the lengths leave to no request, or to a place before its first, are refused;
    those beside them are appended, and nothing else is written."""
    import torch
    from apeiron_b200.step import KV4Cache, SeqBatch

    rng = np.random.default_rng(5)
    k = gpu(rng.standard_normal((6, 1, 64)).astype(np.float32))
    cache = KV4Cache.empty(8, 1, 64, 16)
    cache.pages.fill_(0x11)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = np.arange(8, dtype=np.int32).reshape(2, 4)
    batch = SeqBatch(torch.tensor(cu, **i32), torch.tensor(kv_len, **i32), gpu(table), 6, 6)
    status = ops.new_status()
    ops.rope_kv4_append(None, k, k, ops.rope_table(64, 64), cache, batch, rot_dim=64, status=status)
    assert ops.check_status(status) == (first, 20)
    pages = cache.pages.cpu().numpy()
    right = KV4Cache.empty(8, 1, 64, 16)
    right.pages.fill_(0x11)
    for s in range(2):
        for t in range(cu[s], cu[s + 1]):
            pos = kv_len[s] - cu[s + 1] + t
            if pos >= 0:
                one = SeqBatch(torch.tensor([0, 1], **i32), torch.tensor([pos + 1], **i32),
                               gpu(table[s: s + 1]), 1, 1)
                ops.rope_kv4_append(None, k[t: t + 1], k[t: t + 1], ops.rope_table(64, 64), right,
                                    one, rot_dim=64)
    assert np.array_equal(pages, right.pages.cpu().numpy())
