"""How the dense products are cut up, asked of the plan itself on the CPU: the sizes that the GPU tests run take
every tile in every way of cutting k that ordinary sizes reach, so that a new constant of the plan cannot take
one out of the tests unseen."""
from __future__ import annotations

import subprocess

import pytest

from tests._dense_sizes import FFN, MXFP4
from xkernels_amd import build

MAIN = """
#include <cstdio>
#include <cstdlib>
#include "dense_tile.h"
int main(int n, char** v) {
  for (int i = 1; i + 4 < n; i += 5) {
    const xk::dense::Plan p = xk::dense::plan_tiles(atoll(v[i]) != 0, atoll(v[i + 1]), atoll(v[i + 2]), atoll(v[i + 3]),
                                                    atoll(v[i + 4]) != 0);
    printf("%d %d %d %d %lld\\n", p.rows, p.cols, p.full, p.slices, (long long)p.rest);
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """``plan([(fp4, M, N, chunks, paired), ...])``: for each the tile and the cut of k."""
    d = tmp_path_factory.mktemp("plan")
    (d / "main.hip").write_text(MAIN)
    subprocess.run([build.hipcc(), f"--offload-arch={build.ARCH}", "--offload-host-only", "-std=c++17", "-I",
                    str(build.ROOT / "include"), "-I", str(build.CSRC), str(d / "main.hip"), "-o", str(d / "main")],
                   check=True, capture_output=True)

    def ask(products):
        out = subprocess.run([str(d / "main"), *(str(int(v)) for p in products for v in p)], check=True,
                             capture_output=True, text=True).stdout
        kinds = []
        for line in out.splitlines():
            rows, cols, full, slices, rest = map(int, line.split())
            deep = "" if rows != 128 else " deep" if full + rest * slices <= 256 else " two"
            kinds.append((f"{rows} x {cols}{deep}", "whole" if slices == 1 else "all cut" if full == 0 else "rest cut"))
        assert len(kinds) == len(products)
        return kinds

    return ask


def _ffn(M, H, I):
    """The six products of a step; both weights' gradients are one kernel."""
    def up(n, m):
        return -(-n // m)

    def k(n):  # rows of k are filled up to a multiple of 8
        return up(up(n, 8) * 8, 64)

    return {"gate": [(0, M, I, k(H), 1)], "down": [(0, M, H, k(I), 0)], "dh": [(0, M, I, k(H), 0)],
            "dx": [(0, M, H, k(2 * I), 0)], "dw": [(0, 2 * I, H, up(M, 64), 0), (0, H, I, up(M, 64), 0)]}


SMALL = {("128 x 128 deep", "whole"), ("128 x 128 deep", "all cut"), ("128 x 128 two", "whole"),
         ("128 x 128 two", "all cut"), ("128 x 128 two", "rest cut")}
WIDE = {("256 x 256", "whole"), ("256 x 256", "rest cut"), ("256 x 224", "whole")}
REACHED = {
    "gate": SMALL | {("256 x 256", "whole"), ("256 x 256", "all cut"), ("256 x 256", "rest cut")},
    "down": SMALL | WIDE,
    "dh": SMALL | WIDE | {("256 x 224", "all cut")},
    "dx": SMALL | WIDE | {("256 x 256", "all cut"), ("256 x 224", "all cut")},
    "dw": SMALL | WIDE | {("256 x 256", "all cut"), ("256 x 224", "all cut"), ("256 x 224", "rest cut")},
}


def test_feed_forward_sizes_take_every_tile(plan):
    for name, want in REACHED.items():
        assert set(plan([p for size in FFN for p in _ffn(*size)[name]])) == want, name


def test_mxfp4_sizes_take_every_tile(plan):
    kinds = plan([(1, M, N, -(-(-(-K // 32)) // 8), 0) for M, K, N in MXFP4])
    assert set(kinds) == SMALL - {("128 x 128 two", "all cut")} | WIDE | {("256 x 224", "rest cut")}
    for tile in {t for t, _ in kinds}:  # with whole tiles alone, and with some that pass the output's edges
        rows, cols = int(tile.split()[0]), int(tile.split()[2])
        edges = {M % rows == 0 and N % cols == 0 for (M, _, N), (t, _) in zip(MXFP4, kinds) if t == tile}
        assert edges == {True, False}, tile
