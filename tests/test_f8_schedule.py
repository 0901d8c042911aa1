"""The order of LDS reads, writes and barriers in a step of the weight gradient, walked on the CPU.

The kernel takes the groups in which it reads, stages and waits from f8_wgrad_schedule.h; a host program
prints them for every tile, and the rules that keep two waves of a workgroup from meeting in a buffer are checked on them.
"""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "compute_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "f8_wgrad_schedule.h"
template <class T> void walk(const char* name) {
  for (int q = 0; q < T::kGroups; ++q) {
    const int part = q / T::kPart;
    if (q == T::kBarrier) std::printf("%s %d barrier 0 0\n", name, q);
    // dy operand q + kLast: of the present step or the next
    if (q + T::kLast < T::kGroups) std::printf("%s %d read_dy cur %d\n", name, q, q + T::kLast);
    else std::printf("%s %d read_dy next %d\n", name, q, q + T::kLast - T::kGroups);
    // x operand (run of 16 tokens, t)
    if (part + 1 < T::kParts && q % T::kPart < T::kXGroups)
      for (int e = 0; e < T::kXPer; ++e) {
        const int t = q % T::kPart * T::kXPer + e;
        if (t < T::TK) std::printf("%s %d read_x cur %d\n", name, q, (part + 1) * T::TK + t);
      }
    if (q >= T::kGroups - T::kNextGroups)
      for (int e = 0; e < T::kNextPer; ++e) {
        const int t = (q - (T::kGroups - T::kNextGroups)) * T::kNextPer + e;
        if (t < T::TK) std::printf("%s %d read_x next %d\n", name, q, t);
      }
    if (q >= T::kStageFrom && q < T::kBarrier)
      for (int e = 0; e < T::kPerGroup; ++e) {
        const int p = (q - T::kStageFrom) * T::kPerGroup + e;
        if (p < T::kPieces) std::printf("%s %d stage next %d\n", name, q, p);
      }
    for (int t = 0; t < T::TK; ++t) std::printf("%s %d use_x cur %d\n", name, q, part * T::TK + t);
    std::printf("%s %d use_dy cur %d\n", name, q, q);
  }
  std::printf("%s %d shape %d %d\n", name, T::kGroups, T::kPieces, T::kParts * T::TK);
}
int main() {
  using namespace mx::f8;
  walk<WGradTile256>("bf16_256");
  walk<WGradTile128>("bf16_128");
  walk<WGradTile256F32>("f32_256");
  walk<WGradTile128F32>("f32_128");
}
"""


@pytest.fixture(scope="module")
def steps(tmp_path_factory):
    """{tile: (events of a step in order, groups, pieces staged, x operands)}; an event is (what, which buffer, number)."""
    d = tmp_path_factory.mktemp("schedule")
    (d / "walk.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(d / "walk.cpp"), "-o", str(d / "walk")], check=True)
    out = {}
    for line in subprocess.run([str(d / "walk")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, group, what, buf, number = line.split()
        events, shape = out.setdefault(name, ([], []))
        if what == "shape":
            shape.extend([int(group), int(buf), int(number)])
        else:
            events.append((what, buf, int(number)))
    return {n: (e, *s) for n, (e, s) in out.items()}


TILES = ["bf16_256", "bf16_128", "f32_256", "f32_128"]


@pytest.mark.parametrize("tile", TILES)
def test_no_buffer_is_read_behind_the_barrier_that_frees_it(steps, tile):
    """The next step fills the present buffer from its first group on, and a wave that has passed the barrier may be there."""
    events, *_ = steps[tile]
    at = [what for what, _, _ in events].index("barrier")
    assert [e for e in events[at:] if e[0].startswith("read") and e[1] == "cur"] == []
    assert [e for e in events[:at] if e[0].startswith("read") and e[1] == "next"] == []
    assert [e for e in events[at:] if e[0] == "stage"] == []


@pytest.mark.parametrize("tile", TILES)
def test_every_operand_is_read_once_and_before_its_use(steps, tile):
    events, groups, pieces, x_operands = steps[tile]
    assert [what for what, _, _ in events].count("barrier") == 1
    assert sorted(n for what, _, n in events if what == "stage") == list(range(pieces))
    two = [(w, "cur" if b == "cur" else "next", n, s) for s in (0, 1) for w, b, n in events]
    for kind, count in (("x", x_operands), ("dy", groups)):
        read = {}
        for i, (w, b, n, s) in enumerate(two):
            if w == f"read_{kind}":
                key = (s if b == "cur" else s + 1, n)  # the step it belongs to
                assert key not in read
                read[key] = i
        # the second step's operands: from the first step's end and from its own
        assert {n for s, n in read if s == 1} == set(range(count))
        for i, (w, _, n, s) in enumerate(two):
            if w == f"use_{kind}" and s == 1:
                assert read[1, n] < i
