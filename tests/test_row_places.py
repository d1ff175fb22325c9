"""Which rows share places in memory (csrc/row_places.h), against going through every element."""
import itertools
import os
import random
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = """
#include <cstdio>
#include "row_places.h"
using namespace cudalm_hip;
int main() {
  static uint16_t memory[1];
  long long x[11];
  for (;;) {
    for (auto& v : x) if (std::scanf("%lld", &v) != 1) return 0;
    RowGrid a = {memory, x[0], x[1], x[2], x[3], x[4]};
    RowGrid b = {reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(memory) + 2 * x[10]), x[5], x[6], x[7], x[8], x[9]};
    std::printf("%d %d %d\\n", places_apart(a), places_meet(a, b), places_meet(b, a));
  }
}
"""


def _run(tmp_path, rows):
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = str(tmp_path / "main")
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(REPO, "cudalm-agent_amd", "csrc"),
                          str(tmp_path / "main.cpp"), "-o", exe], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([exe], input="\n".join(" ".join(map(str, r)) for r in rows), capture_output=True, text=True,
                         timeout=120).stdout
    return [tuple(int(x) for x in line.split()) for line in out.splitlines()]


def _places(count, step, side, between, width, at=0):
    return [at + i * step + j * between + e for i in range(count) for j in range(side) for e in range(width)]


def test_against_every_element(tmp_path):
    rng = random.Random(5)
    rows = []
    for _ in range(6000):
        n, side_a, side_b = rng.randint(1, 6), rng.randint(1, 5), rng.randint(1, 5)
        step, between = rng.randint(-20, 20), rng.randint(-20, 20)
        wa, wb = rng.randint(1, 5), rng.randint(1, 5)
        rows.append((n, step, side_a, between, wa, n, step, side_b, between, wb, rng.randint(-60, 60)))
    both = [0, 0]
    for r, (apart, meet, back) in zip(rows, _run(tmp_path, rows)):
        a, b = _places(*r[:5]), _places(*r[5:10], at=r[10])
        assert apart == (len(set(a)) == len(a)), r
        assert meet == back == bool(set(a) & set(b)), r
        both[meet] += 1
    assert min(both) > 500


def test_layouts_of_tensors(tmp_path):
    """Queries, keys and values side by side; heads outside; columns of one tensor; other strides."""
    apart = [(5, 12 * 64, 8, 64, 64, 5, 12 * 64, 2, 64, 64, 8 * 64), (5, 64, 8, 5 * 64, 64, 5, 64, 2, 5 * 64, 64, 40 * 64),
             (30, 90, 1, 0, 48, 30, 90, 1, 0, 30, 49), (3, 10, 2, 5, 5, 3, 11, 2, 5, 5, 0),
             (2 ** 31 - 1, 2 ** 40, 2 ** 22, 2 ** 15, 2 ** 15, 2 ** 31 - 1, 2 ** 40, 1, 7, 8, 2 ** 38)]
    for r, got in zip(apart, _run(tmp_path, apart)):
        assert got == (1, 0, 0), r
    # one place for two rows of two heads; the third head at the next token; a view one element on
    for r, want in (((2, 64, 2, 64, 64, 2, 64, 2, 64, 64, 10 ** 6), 0), ((2, 128, 3, 64, 64, 2, 128, 3, 64, 64, 10 ** 6), 0),
                    ((30, 90, 1, 0, 48, 30, 90, 1, 0, 30, 47), 1)):
        got = _run(tmp_path, [r])[0]
        assert got[0] == want and got[1:] == (want, want), r
    # one row each: strides mean nothing
    for at, (x, y) in itertools.product((39, 40), [(1, 9)]):
        assert _run(tmp_path, [(1, x, 1, 3, 40, 1, y, 1, 4, 8, at)])[0] == (1, at < 40, at < 40)
