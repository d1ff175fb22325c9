"""Where the join of attention with shared prefixes reads (csrc/paged_places.h), for entries that
are written and for ones that hold anything: the memory of a workspace, where lengths change under a call."""
import os
import random
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = """
#include <cstdio>
#include "paged_places.h"
using namespace cudalm_hip;
int main() {
  int x[8];
  for (;;) {
    for (auto& v : x) if (std::scanf("%d", &v) != 1) return 0;
    const SegmentParts p = parts_within({x[0], x[1], x[2], x[3]}, x[4], x[5], x[6], x[7]);
    int least = p.first, most = p.first;
    for (int y = 0; y < p.own; ++y) {
      const int at = own_part(p.first, y);
      least = at < least ? at : least, most = at > most ? at : most;
    }
    std::printf("%d %d %d %d %d %d\\n", p.first, p.own, p.prefix, p.row, least, most);
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


def test_entries_of_calls(tmp_path):
    """Segments cut into ranges as the kernel cuts them: what it writes stays as it is."""
    rng = random.Random(2)
    rows = []
    for _ in range(300):
        segments, ranges, splits = rng.randint(1, 9), rng.randint(1, 12), rng.randint(1, 5)
        counts = [rng.randint(1, 30) for _ in range(segments)]
        per, g = -(-sum(counts) // ranges), 0
        r = rng.randint(1, 40)
        prefix_rows = 128 * (segments * r // 128 + 1)
        for s, n in enumerate(counts):
            first, last = g // per, (g + n - 1) // per
            slot = 2 * ranges + s if first == last else 2 * first + 1
            rows.append((slot, last - first + 1, rng.randint(0, splits), rng.randint(0, prefix_rows - r), 2 * ranges + segments,
                         splits, prefix_rows, r))
            g += n
    for row, got in zip(rows, _run(tmp_path, rows)):
        assert got[:4] == row[:4] and got[5] < row[4], row


def test_entries_that_hold_anything(tmp_path):
    rng = random.Random(3)
    any_int = lambda: rng.choice([rng.randint(-2 ** 31, 2 ** 31 - 1), rng.randint(-5, 60), -2 ** 31, 2 ** 31 - 1])  # noqa: E731
    rows = []
    for _ in range(4000):
        r = rng.randint(1, 1024)
        rows.append((any_int(), any_int(), any_int(), any_int(), rng.randint(1, 50), rng.randint(1, 9),
                     128 * rng.randint(9, 40), r))
    for row, (first, own, prefix, at, least, most) in zip(rows, _run(tmp_path, rows)):
        slots, splits, prefix_rows, r = row[4:]
        assert 0 <= least and most < slots, row
        assert 0 <= prefix <= splits and 0 <= at and at + r <= prefix_rows, row
