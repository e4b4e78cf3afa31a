"""CPU test of how a K split of the 8-bit products deals out k blocks and the
units in which their scales come (linear8.cuh): what is fetched is what the
blocks use, so that no load is left in flight when a CTA leaves."""
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
SOURCE = r'''
#include <cstdio>
#include "linear8.cuh"
int main() {
  for (int blocks = 1; blocks <= 40; ++blocks)
    for (int split = 1; split <= 4; ++split)
      for (int rank = 0; rank < split; ++rank) {
        const senmoe::KRange k = senmoe::k_share(blocks, rank, split), u = senmoe::scale_units(k.begin, k.end);
        printf("%d %d %d %d %d %d %d\n", blocks, split, rank, k.begin, k.end, u.begin, u.end);
      }
}
'''


@pytest.fixture(scope="module")
def ranges(tmp_path_factory):
    import build
    d = tmp_path_factory.mktemp("ranges")
    (d / "t.cu").write_text(SOURCE)
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", build.CSRC, "-I", build.INCLUDE,
                    str(d / "t.cu"), "-o", str(d / "t")], check=True)
    out = subprocess.run([str(d / "t")], capture_output=True, text=True, check=True).stdout
    return [tuple(int(v) for v in line.split()) for line in out.splitlines()]


def test_k_blocks_are_dealt_out_once(ranges):
    held = {}
    for blocks, split, rank, k0, k1, _, _ in ranges:
        held.setdefault((blocks, split), []).extend(range(k0, k1))
    assert held and all(v == list(range(blocks)) for (blocks, _), v in held.items())


def test_scale_units_are_those_of_the_blocks(ranges):
    for blocks, split, rank, k0, k1, u0, u1 in ranges:
        assert list(range(u0, u1)) == sorted({b // 2 for b in range(k0, k1)}), (blocks, split, rank)


def test_planning_takes_no_longer_with_more_rows():
    """The choice of tiles for a grouped product, on the host before every launch.  The K split is refused for so many
    tiles, after the choice and before anything is launched."""
    import ctypes as C
    import time

    import build
    build.build()
    import senmoe
    P = 0x10000  # never read
    q = senmoe.SenMoeLinear8(dtype=0, epilogue=0, num_groups=2, path=senmoe.LINEAR_TCGEN05_SPLIT, rows=(1 << 31) - 1024,
                             in_features=64, out_features=16, x=P, x_stride=64, x_scales=P, x_scales_stride=2, weight=P,
                             weight_stride=64, weight_group_stride=1024, weight_scales=P, weight_scales_stride=2,
                             weight_scales_group_stride=32, offsets=P, y=P, y_stride=16)
    took = []
    for _ in range(3):
        start = time.perf_counter()
        assert senmoe.lib().senmoe_linear8(C.byref(q), None) == 5
        took.append(time.perf_counter() - start)
    assert min(took) < 0.01, took  # (a few microseconds; seconds where every chunk of 2^30 rows is counted)
