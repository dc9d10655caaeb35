"""CPU check of the tile ring of the drafted tokens' tensor-core kernel: tests/tree_ring_check.cpp is compiled with g++
against the header that the kernel itself uses (csrc/ex_tree_ring.h) and runs every interleaving of the producer warps and the
consumer on rings of 1 to 3 slots, over tiles with all boxes, with one (a request's tail: most producers have none) and with
none (pages that do not exist). No tile may be read before its boxes are there or written before it was used up, and no
wait may be left that cannot end. A planted variant must fail: one where only the producers with something to announce
arrive, so that a slot can be filled, used up and filled again while a producer without a box stands still, whose wait is
then on the parity of another lap."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_tree_ring_in_every_interleaving(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "tree_ring_check"
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Werror", "-I", str(ROOT / "vllm-exact_b200" / "csrc"),
                    str(ROOT / "tests" / "tree_ring_check.cpp"), "-o", str(exe)], check=True, capture_output=True, text=True,
                   timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    word, runs, planted = r.stdout.split()
    assert word == "OK" and int(runs) == 30 and int(planted) >= 10
