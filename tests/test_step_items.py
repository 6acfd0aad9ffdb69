"""The split of the attention over the 4-bit cache into items and shares, compiled for the host from
the kernel's own header: each step belongs to one item, and what a CTA owes to items that cross its
ends follows from the lengths alone, so that a CTA whose wait has given up still counts itself and
leaves every counter as it found it."""
import os
import subprocess

import pytest

from apeiron_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_items_and_what_ctas_owe(tmp_path):
    exe = str(tmp_path / "attn_items")
    try:
        nvcc = build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    subprocess.run([nvcc, *build.ARCH, "-std=c++17", "-O2", "-I", build.CSRC, "-o", exe,
                    os.path.join(HERE, "attn_items.cu")], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
