"""Which columns of a workgroup see a position, as one range (compiled as plain C++), against the rule position by position."""
from __future__ import annotations

import subprocess

import numpy as np

from opentars_amd import build

TOP = 2 ** 31 - 1


def test_the_columns_that_see_a_position(tmp_path):
    (tmp_path / "range.cpp").write_text(r'''
#include <cstdio>
#include "paged_index.h"
int main() {
  int v[7];
  while (std::scanf("%d %d %d %d %d %d %d", v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6) == 7) {
    const tars::Range r = tars::seen_by(v[0], v[1], v[2], v[3], v[4], v[5], v[6]);
    std::printf("%d %d\n", r.lo, r.hi);
  }
}
''')
    exe = tmp_path / "range"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-Wall", "-Werror",
                    "-I", str(build.CSRC), str(tmp_path / "range.cpp"), "-o", str(exe)], check=True, capture_output=True)
    rng = np.random.default_rng(7)
    cases = []
    for _ in range(20000):
        group, cols = int(rng.choice([1, 2, 3, 8, 40, 200])), int(rng.choice([1, 16, 31, 32, 128, rng.integers(1, 129)]))
        c0 = int(rng.choice([0, 0, 16, 128, 128 * rng.integers(0, 30)]))
        window = int(rng.choice([0, 0, 1, 5, 40, 300, TOP]))
        sinks = int(rng.choice([0, 0, 4, 60, TOP]))
        cases.append((int(rng.integers(0, 400)), int(rng.integers(-60, 350)), group, c0, cols, window, sinks))
    cases += [(2 ** 30 - 1, p0, 64, c0, 128, w, s) for p0 in (-2 ** 22, 2 ** 30 - 2 ** 22, 2 ** 30 - 1) for c0 in (0, 2 ** 28 - 128)
              for w in (0, 1, 2 ** 30, TOP) for s in (0, 7, TOP)]
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    got = np.array([int(x) for x in out.split()]).reshape(-1, 2)
    for (j, p0, group, c0, cols, w, s), (lo, hi) in zip(cases, got.tolist()):
        p = p0 + (c0 + np.arange(cols)) // group
        seen = (j <= p) & ((w == 0) | (j > p - w) | (j < s))
        assert 0 <= lo <= cols and 0 <= hi <= cols
        assert np.array_equal(seen, (np.arange(cols) >= lo) & (np.arange(cols) < hi)), (j, p0, group, c0, cols, w, s)
