"""Which arrays the kernels reach by 32-bit byte offsets (nerf_amd/csrc/offsets.hpp),
compiled for the host and compared with whole-number arithmetic: every offset that
a kernel forms stays below 2^31, where an access is taken for one beyond the array."""
import itertools
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nerf_amd" / "csrc"
CHUNK = 1024  # positions whose rows are reached from one start without an index
SOURCE = """
#include <cstdio>
#include "offsets.hpp"
using namespace nerf_hip::grouped;
int main() {
    unsigned long long count, widest;
    int index;
    while (std::scanf("%d %llu %llu", &index, &count, &widest) == 3) std::printf("%d %d %u\\n", near(count, widest), stream_outputs_near(index != 0, count, widest), kStreamChunk);
}
"""


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ is required")
    at = tmp_path_factory.mktemp("offsets")
    (at / "main.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++20", "-Wall", "-Wextra", "-Werror", "-I", str(CSRC), str(at / "main.cpp"), "-o", str(at / "main")], check=True)

    def ask(cases):
        out = subprocess.run([str(at / "main")], input="".join(f"{int(i)} {c} {w}\n" for i, c, w in cases), capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return ask


def test_offsets_of_outputs(answers):
    """Rows of up to 2^20 values of 16 or (as twice as many) 32 bits, up to 2^30 of them."""
    widths = [8, 256, 2**19, 2**20 - 8, 2**20 - 4, 2**20, 2**20 + 8, 2**21 - 8, 2**21]
    counts = [1, 1023, 1024, 1025, 65536, 2**22, 2**30]
    cases = list(itertools.product((False, True), counts, widths))
    for (index, count, wide), (near, outputs, chunk) in zip(cases, answers(cases)):
        assert chunk == CHUNK
        end = 2 * wide * count  # the bytes of `count` rows
        assert bool(near) == (end < 2**31), (count, wide)
        # The last byte that is reached, counted from an index' array or a chunk's first row.
        last = 2 * wide * (count if index else CHUNK) - 1
        assert not outputs or last < 2**31, (index, count, wide)
        assert outputs or 2 * wide * (count if index else CHUNK) >= 2**31, (index, count, wide)


def test_the_widest_rows_without_an_index(answers):
    """fp32 outputs 2^19 values apart: row 1023 of a chunk starts 2^31 - 2^21 bytes from
    its first, and 2^20 values apart beyond 32 bits."""
    assert [a[1] for a in answers([(False, 65536, 2 * 2**19), (False, 65536, 2 * 2**20), (False, 65536, 2 * (2**19 - 8))])] == [0, 0, 1]
