"""The embedding's kernels from their own source on the CPU, a work-item at a time (tests/waves): every buffer lies between pages that
cannot be touched, the list of tokens by id is checked entry by entry, and sums of whole numbers are compared exactly."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from torchure_amd import build_native

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "waves")
CSRC = os.path.join(build_native.ROOT, "torchure_amd", "csrc")


def clang() -> str:
    for cand in ("/opt/rocm/llvm/bin/clang++", shutil.which("amdclang++"), shutil.which("clang++")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("clang++ not found")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("waves") / "embed")
    subprocess.run([clang(), "-O2", "-std=c++17", "-w", f"-I{HERE}", f"-I{build_native.INCLUDE}", f"-I{CSRC}", "-x", "c++",
                    os.path.join(HERE, "embed.cpp"), os.path.join(HERE, "waves.cpp"), "-o", out], check=True)
    return out


# tokens, ids of the table, columns, which ids, padding, added to a table, 64-bit ids, table fp32, gradient fp32, elements between rows
@pytest.mark.parametrize("args", [
    (1, 1, 1, "any", -1, 0, 1, 1, 1, 0),
    (1, 5, 9, "outside", -1, 1, 0, 0, 0, 3),
    (32, 3, 7, "same", -1, 0, 1, 0, 1, 1),
    (33, 3, 8, "same", 1, 1, 1, 1, 0, 0),
    (64, 300, 257, "any", -1, 1, 1, 1, 1, 5),
    (65, 2, 12, "text", 1, 0, 0, 0, 0, 2),
    (500, 300, 777, "text", 3, 0, 1, 0, 0, 0),
    (500, 300, 520, "outside", 7, 1, 0, 1, 0, 1),
    (700, 40, 16, "padding", 5, 0, 1, 0, 0, 0),
    (700, 40, 16, "padding", 5, 1, 0, 1, 1, 0),
    (1025, 8193, 3, "text", -1, 1, 1, 0, 1, 0),
    (2049, 1, 4, "same", -1, 0, 1, 1, 1, 0),  # more of an id than wait at once, in one part and in several
    (4097, 2, 40, "text", -1, 0, 0, 0, 0, 1),
    (8193, 1, 5, "any", -1, 1, 1, 0, 0, 0),
    (20000, 300, 4, "text", 299, 0, 1, 1, 0, 0),
    (3000, (1 << 21) + 5, 1, "any", -1, 1, 1, 1, 1, 0),  # more ids than 256 workgroups hold
    (50001, 4096, 777, "text", 3, 0, 1, 0, 0, 0),
])
def test_every_access_and_sum(program, args):
    done = subprocess.run([program, *map(str, args)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.endswith("ok\n"), (done.returncode, done.stdout[-500:], done.stderr[-500:])
