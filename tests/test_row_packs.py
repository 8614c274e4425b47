"""Rows that a block's threads share out, on the CPU (row_packs.cu): every place comes once, for rows so wide that
their places together pass 32 bits too."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def places(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("row_packs") / "row_packs")
    subprocess.check_call([shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17",
                           "-I", os.path.join(PKG_DIR, "csrc"), "-I", os.path.join(ROOT, "include"), os.path.join(HERE, "row_packs.cu"), "-o", exe])

    def run(begin, end, rows, thread):
        most = (end - begin) * rows // 256 + 4096
        out = subprocess.run([exe, *map(str, (begin, end, rows, thread, most))], capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, {1: "more places than there are", 2: "a place outside"}.get(out.returncode, out.returncode)
        return [int(v) for v in out.stdout.split()]
    return run


@pytest.mark.parametrize("begin,end,rows", [(0, 1, 1), (5, 6, 64), (3, 3, 16), (0, 1000, 7), (17, 2065, 64), (9, 300, 33)])
def test_every_place_once(places, begin, end, rows):
    got = [places(begin, end, rows, t) for t in range(256)]
    assert sum(n for n, _ in got) == (end - begin) * rows
    assert sum(s for _, s in got) == sum(r * 3 + p for r in range(rows) for p in range(begin, end))


@pytest.mark.parametrize("begin,end,rows", [(0, 1 << 28, 16), (1 << 28, (1 << 29) + 1, 16), (0, (1 << 26) + 1, 64), (0, (1 << 28) - 100, 16),
                                            ((1 << 30) - (1 << 26) - 77, (1 << 30) - 1, 64)])
def test_rows_whose_places_pass_32_bits(places, begin, end, rows):
    """A block of 16 rows of 2^29 channels, and the like: some 256th of the places for the first and the last thread."""
    whole = (end - begin) * rows
    pieces = -(-(end - begin) // (1 << 24))
    for thread in (0, 255):
        n, _ = places(begin, end, rows, thread)
        assert abs(n - whole // 256) <= pieces + 1
