"""Sizes of launches at the ends of the documented ranges, without a GPU: the host's arithmetic, compiled alone."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "vte_amd" / "csrc"

PROGRAM = """
#include <cstdio>
#include "launch.h"
int main() {
    long long n;
    int wide, hd, size;
    while (std::scanf("%lld %d %d %d", &n, &wide, &hd, &size) == 4) {
        const int per = vte::qk_norm_heads(wide != 0, hd, size);
        const vte::BlockGrid g = vte::block_grid((n + per - 1) / per);
        std::printf("%d %u %u\\n", per, g.x, g.y);
    }
}
"""


@pytest.fixture(scope="module")
def shapes(tmp_path_factory):
    """[(heads of a block, x, y)] of [(heads, wide, head_dim, bytes of a value)]."""
    d = tmp_path_factory.mktemp("launch")
    (d / "m.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(d / "m.cpp"), "-o", str(d / "m")], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(d / "m")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def test_every_accepted_number_of_heads_can_be_launched(shapes):
    """Up to 2^27 heads (rows times heads of q and k), of every form, length and type: below 2^32 threads a dimension, at most
    65535 blocks in the second one, all heads reached, and the last block's numbers are still ints."""
    heads = sorted({n for p in range(28) for n in (2 ** p - 1, 2 ** p, 2 ** p + 1) if 1 <= n <= 2 ** 27})
    cases = [(n, wide, hd, size) for n in heads for wide in (0, 1) for hd in (64, 128, 256) for size in (2, 4)]
    for (n, wide, hd, size), (per, x, y) in zip(cases, shapes(cases), strict=True):
        assert per * hd * size == 8192 if wide else per == 4
        assert 1 <= x and x * 256 < 2 ** 32 and 1 <= y <= 65535, (n, wide, hd, size)
        assert x * y * per >= n and (x * y + 1) * per < 2 ** 31 and (y - 1) * x * per < n
        assert y == 1 or x * per * 2 <= n + x * per


def test_common_sizes_have_one_dimension(shapes):
    assert shapes([(14, 1, 128, 2), (4096 * 32, 1, 128, 4), (4096 * 32, 0, 128, 2)]) == [(32, 1, 1), (16, 8192, 1), (4, 32768, 1)]
