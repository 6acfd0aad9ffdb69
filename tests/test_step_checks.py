"""What apeiron_b200.step refuses before it calls the library, without a GPU: tensors are stood in
for by their attributes."""
import pytest
import torch

from apeiron_b200 import _abi, build
from apeiron_b200.step import DeviceAct, KV4Cache, SeqBatch, StepOps


class Fake:
    """A contiguous tensor on GPU `dev` as the checks see it; nothing reads its memory."""

    def __init__(self, shape, dtype=torch.float32, dev=0, ptr=1 << 20):
        self.shape, self.dtype, self.dev, self.ptr = torch.Size(shape), dtype, dev, ptr
        self.is_cuda, self.device = dev >= 0, torch.device("cuda", dev) if dev >= 0 else None

    def get_device(self):
        return self.dev

    def numel(self):
        return self.shape.numel()

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def stride(self):
        return tuple(self.shape[i + 1:].numel() for i in range(len(self.shape)))

    def data_ptr(self):
        return self.ptr


I32 = torch.int32


@pytest.fixture(scope="module")
def ops():
    """StepOps of GPU 1, whose entry points record that they were reached."""
    class Backend:
        lib, ctx, device = _abi.load(build.build()), None, 1

    ops = StepOps(Backend())
    ops.reached = []
    for name in ("_norm", "_rope", "_attn", "_sample"):
        setattr(ops, name, lambda *a, name=name: ops.reached.append(name) or 0)
    return ops


def cache(dev=1):
    return KV4Cache(Fake((8, 2, KV4Cache.page_bytes(64, 16)), torch.uint8, dev), 2, 64, 16)


def batch(dev=1, table_dev=None, cu_dev=None):
    pick = lambda d: dev if d is None else d  # noqa: E731
    return SeqBatch(Fake((2,), I32, pick(cu_dev)), Fake((1,), I32, dev),
                    Fake((1, 4), I32, pick(table_dev)), 4, 4)


# a call with every tensor it takes; `wrong` is the one that is on another GPU (or on none)
def norm(ops, on):
    ops.add_rms_norm_quant(on("x", (4, 64)), on("weight", (64,)), 1e-6, add=on("add", (4, 64)),
                           resid=on("resid", (4, 64)), y=on("y", (4, 64)),
                           deq=on("deq", (4, 64)), stream=0)


def rope(ops, on):
    f16 = torch.float16
    ops.rope_kv4_append(on("q", (4, 4, 64)), on("k", (4, 2, 64)), on("v", (4, 2, 64)),
                        on("table", (16, 32, 2)), cache(), batch(), rot_dim=64,
                        q_out=on("q_out", (4, 4, 64)), k_deq=on("k_deq", (4, 2, 64), f16),
                        v_deq=on("v_deq", (4, 2, 64), f16),
                        status=on("status", (2,), torch.int64), stream=0)


def attn(ops, on):
    ops.attn_kv4(on("q", (4, 4, 64)), cache(), batch(), 1.0, out=on("out", (4, 4, 64)),
                 status=on("status", (2,), torch.int64), stream=0)


def sample(ops, on):
    ops.sample(on("logits", (3, 10)), on("u", (3,)), temperature=on("temperature", (3,)),
               top_k=on("top_k", (3,), I32), top_p=on("top_p", (3,)), min_p=on("min_p", (3,)),
               token=on("token", (3,), I32), prob=on("prob", (3,)), kept=on("kept", (3,), I32),
               stream=0)


@pytest.mark.parametrize("call", [norm, rope, attn, sample])
def test_tensors_of_another_gpu(ops, call):
    names = []

    def all_here(name, shape, dtype=torch.float32):
        names.append(name)
        return Fake(shape, dtype, 1)

    ops.reached.clear()
    call(ops, all_here)
    assert len(ops.reached) == 1
    for wrong in names:
        for dev in (0, -1):
            with pytest.raises(ValueError):
                call(ops, lambda name, shape, dtype=torch.float32: Fake(
                    shape, dtype, dev if name == wrong else 1))
    assert len(ops.reached) == 1


def test_caches_and_batches_of_another_gpu(ops):
    q, k = Fake((4, 4, 64), dev=1), Fake((4, 2, 64), dev=1)
    table = Fake((16, 32, 2), dev=1)
    ops.reached.clear()
    for c, b in ((cache(0), batch()), (cache(), batch(0)), (cache(0), batch(0))):
        with pytest.raises(ValueError):
            ops.attn_kv4(q, c, b, 1.0, out=Fake((4, 4, 64), dev=1), stream=0)
        with pytest.raises(ValueError):
            ops.rope_kv4_append(None, k, k, table, c, b, rot_dim=64, stream=0)
    assert not ops.reached
    for kw in (dict(table_dev=0), dict(cu_dev=0), dict(dev=-1)):
        with pytest.raises(ValueError):
            batch(**kw)


def test_activations_of_the_wrong_size(ops):
    """A DeviceAct from a caller's own tensors holds what the kernels write."""
    pad = ops.lib.apx_act_padded_len(100)
    right = dict(codes=Fake((3, pad), torch.int8, 1), exps=Fake((3, pad // 32), torch.uint8, 1),
                 descs=Fake((3, 8), I32, 1))
    x = Fake((3, 100), dev=1)
    act = DeviceAct(**right, n=100)
    ops.reached.clear()
    assert ops.add_rms_norm_quant(x, None, 1e-6, act=act, stream=0) is act
    assert ops.reached == ["_norm"]
    for name, wrong in (
            ("codes", Fake((3, 100), torch.int8, 1)), ("codes", Fake((3, pad), torch.uint8, 1)),
            ("codes", Fake((3, pad), torch.int8, -1)), ("codes", Fake((3 * pad,), torch.int8, 1)),
            ("exps", Fake((3, pad // 32 - 1), torch.uint8, 1)), ("exps", Fake((3, pad), torch.int8, 1)),
            ("exps", Fake((3, pad // 32), torch.uint8, 0)),
            ("descs", Fake((3, 4), I32, 1)), ("descs", Fake((2, 8), I32, 1)),
            ("descs", Fake((3, 8), torch.int64, 1))):
        with pytest.raises(ValueError):
            DeviceAct(**{**right, name: wrong}, n=100)
    other = DeviceAct(**{k: Fake(t.shape, t.dtype, 0) for k, t in right.items()}, n=100)
    with pytest.raises(ValueError):
        ops.add_rms_norm_quant(x, None, 1e-6, act=other, stream=0)
    with pytest.raises(ValueError):  # of 100 lanes for rows of 99
        ops.add_rms_norm_quant(Fake((3, 99), dev=1), None, 1e-6, act=act, stream=0)
    assert ops.reached == ["_norm"]


def test_numbers_that_no_field_holds(ops):
    """Numbers past the C structs' fields are refused as other arguments are, not cut to them."""
    q, k = Fake((4, 4, 64), dev=1), Fake((4, 2, 64), dev=1)
    table = Fake((16, 32, 2), dev=1)
    ops.reached.clear()
    for kw in (dict(window=2 ** 31), dict(window=2 ** 63), dict(sinks=2 ** 31), dict(window=3.5)):
        with pytest.raises(ValueError):
            ops.attn_kv4(q, cache(), batch(), 1.0, out=q, stream=0, **kw)
    for rot in (2 ** 31, 2 ** 32 + 64):
        with pytest.raises(ValueError):
            ops.rope_kv4_append(None, k, k, table, cache(), batch(), rot_dim=rot, stream=0)
    for n_pos, rot in ((-1, 64), (4, -8), (4, 2 ** 32 + 64), (2 ** 32, 64)):
        with pytest.raises(ValueError):
            ops.rope_table(n_pos, rot, stream=0)
    assert not ops.reached
    i32 = lambda *s: Fake(s, I32, 1)  # noqa: E731
    for n, most in ((2 ** 32 + 4, 4), (4, 2 ** 32 + 4), (-1, 4), (4, -1)):
        with pytest.raises(ValueError):
            SeqBatch(i32(2), i32(1), i32(1, 4), n, most)
    pages = Fake((8, 2, KV4Cache.page_bytes(64, 16)), torch.uint8, 1)
    for dim, tokens in ((2 ** 32 + 64, 16), (64, 2 ** 32 + 16), (64, -16)):
        with pytest.raises(ValueError):
            KV4Cache(pages, 2, dim, tokens)


def test_calls_on_a_closed_backend():
    """A backend that was closed has no context: the entry points get none, and refuse."""
    class Backend:
        lib, ctx, device = _abi.load(build.build()), 77, 1

    ops = StepOps(Backend())
    given = []
    names = ("_norm", "_rope", "_attn", "_sample")
    for name in names:
        setattr(ops, name, lambda ctx, *a: given.append(ctx) or 0)
    here = lambda name, shape, dtype=torch.float32: Fake(shape, dtype, 1)  # noqa: E731
    for call in (norm, rope, attn, sample):
        call(ops, here)
    ops.backend.ctx = None  # as Backend.close leaves it
    for call in (norm, rope, attn, sample):
        call(ops, here)
    assert given == [77] * 4 + [None] * 4 and ops.ctx is None
    real = StepOps(ops.backend)
    for call in (norm, rope, attn, sample):
        with pytest.raises(ValueError):
            call(real, here)
