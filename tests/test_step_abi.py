"""The C structs of the steps between the projections and their ctypes mirrors, and what the entry
points refuse without a device."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from apeiron_b200 import _abi, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("mirror,name", [
    (_abi.NormArgs, "apx_norm_args"), (_abi.Kv4Cache, "apx_kv4_cache"),
    (_abi.SeqBatch, "apx_seq_batch"), (_abi.RopeFreqs, "apx_rope_freqs"),
    (_abi.RopeArgs, "apx_rope_args"), (_abi.AttnArgs, "apx_attn_args"),
    (_abi.SampleArgs, "apx_sample_args")])
def test_struct_layouts_match_the_header(tmp_path, mirror, name):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [f for f, _ in mirror._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "apeiron_cuda.h"\n'
                   f'int main(void) {{\n  printf("%zu\\n", sizeof({name}));\n' +
                   "".join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) +
                   "  return 0;\n}\n")
    exe = tmp_path / "probe"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert out == [C.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


def test_packed_arguments_have_the_structs_layout():
    """apeiron_b200.step packs each call's arguments in one go: the mirrors' size and offsets."""
    from apeiron_b200 import step

    for pack, mirror in ((step._NORM, _abi.NormArgs), (step._ROPE, _abi.RopeArgs),
                         (step._ATTN, _abi.AttnArgs), (step._SAMPLE, _abi.SampleArgs)):
        kinds = [t for _, t in mirror._fields_]
        values = [0.5 + i if t is C.c_float else 3 + i for i, t in enumerate(kinds)]
        raw = pack(*values)
        assert len(raw) == C.sizeof(mirror)
        got = mirror.from_buffer_copy(raw)
        assert [getattr(got, f) for f, _ in mirror._fields_] == values


@pytest.fixture(scope="module")
def lib():
    return _abi.load(build.build())


def test_page_bytes(lib):
    """9/16 byte a value (4 bits, and 16 bits of scale for 32 of them), K and V."""
    for dim in (64, 128):
        for page in (16, 32, 64, 128):
            assert lib.apx_kv4_page_bytes(dim, page) == 2 * page * dim * 9 // 16
    for dim, page in ((0, 16), (96, 16), (256, 16), (64, 8), (64, 48), (64, 256), (-64, 16)):
        assert lib.apx_kv4_page_bytes(dim, page) == 0


def test_no_context_is_refused(lib):
    cache, batch = _abi.Kv4Cache(), _abi.SeqBatch()
    bad = _abi.APX_ERR_INVALID_ARGUMENT
    assert lib.apx_add_rms_norm_quant_async(None, C.byref(_abi.NormArgs()), None) == bad
    assert lib.apx_rope_table_async(None, C.byref(_abi.RopeFreqs()), 1, None, None) == bad
    assert lib.apx_rope_kv4_append_async(None, C.byref(_abi.RopeArgs()), C.byref(cache),
                                         C.byref(batch), None) == bad
    assert lib.apx_attn_kv4_async(None, C.byref(_abi.AttnArgs()), C.byref(cache), C.byref(batch),
                                  None) == bad
    assert lib.apx_sample_async(None, C.byref(_abi.SampleArgs()), None) == bad
