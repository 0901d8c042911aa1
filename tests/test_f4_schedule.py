"""The loads of scales of w [N, K] in the product over 4-bit blocks on the bf16 matrix cores, walked on the CPU.

The kernel takes from f4_wide_schedule.h which bytes of a row a load begins with, with which step's codes it goes, and where a
step's scales are read; a host program prints them for every slice that K could be cut into.
"""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "compute_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "f4_wide_schedule.h"
int main(int, char** v) {
  using namespace mx::f4;
  const int s0 = std::atoi(v[1]), s1 = std::atoi(v[2]), buffers = std::atoi(v[3]);
  std::printf("load 0 %d %d\n", scales_at(s0, 0), s0);
  for (int s = s0; s < s1 + buffers; ++s)
    if (const int t = scales_with(s, s0, buffers)) std::printf("load %d %d %d\n", t, scales_at(s0, t), s);
  for (int s = s0; s < s1; ++s) std::printf("read %d %d %d\n", scales_group(s, s0), scales_byte(s, s0), s);
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("schedule")
    (d / "walk.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(d / "walk.cpp"), "-o", str(d / "walk")], check=True)

    def run(s0, s1, buffers):
        """([(group, byte of the row, the step whose codes it goes with)], [(group, byte of the group, step)])"""
        lines = subprocess.run([str(d / "walk"), str(s0), str(s1), str(buffers)], check=True, capture_output=True, text=True).stdout.split("\n")
        events = [(w[0], tuple(map(int, w[1:]))) for w in map(str.split, lines) if w]
        return [e for w, e in events if w == "load"], [e for w, e in events if w == "read"]

    return run


def slices_of(K):
    steps = K // 64
    for S in range(1, min(steps, 16) + 1):
        per = -(-steps // S)
        for s0 in range(0, steps, per):
            yield s0, min(steps, s0 + per)


SLICES = sorted({s for K in (128, 256, 384, 1280, 1536, 2560, 4096, 5120) for s in slices_of(K)})


@pytest.mark.parametrize("buffers", [2, 3, 4])  # those of the tiles
def test_scales_of_every_slice(walk, buffers):
    for s0, s1 in SLICES:
        loads, reads = walk(s0, s1, buffers)
        where = {}
        for t, at, step in loads:
            assert at % 4 == 0, (s0, s1)  # a load's words are words of the row: each inside the array or outside it
            assert t not in where
            where[t] = (at, step)
        for t, byte, step in reads:
            at, requested = where[t]
            assert at + byte == 2 * step and byte < 16, (s0, s1, step)  # the step's own scales
            assert requested <= step, (s0, s1, step)  # arrived behind the barrier before the step
        last = {t: max(s for g, _, s in reads if g == t) for t, _, _ in reads}
        for t, (_, requested) in where.items():  # the buffer's group before it has been read
            if t >= 2:
                assert requested - buffers >= last[t - 2], (s0, s1, t)
            else:
                assert t == 0 or requested >= s0


def test_odd_slices_are_among_them():
    """64 steps in six slices of 11, 40 in eight of five: slices that the plans of 17 rows take."""
    assert {(11, 22), (55, 64), (5, 10), (35, 40)} <= set(SLICES)
