"""The reads of a list of page copies, walked on the host as the copy kernel walks it."""
from __future__ import annotations

import random
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "page_runs.cuh"
int main() {
  int n;
  while (scanf("%d", &n) == 1) {
    std::vector<int32_t> src(n), dst(n);
    for (auto& x : src) if (scanf("%d", &x) != 1) return 1;
    for (auto& x : dst) if (scanf("%d", &x) != 1) return 1;
    for (int64_t i = 0; i < n; ++i) {
      int64_t j = gdn::run_first(src.data(), dst.data(), n, i);
      if (j < 0) continue;
      printf("r %d\n", src[i]);
      for (; j >= 0; j = gdn::run_next(src.data(), n, j))
        if (dst[j] >= 0) printf("w %d %d\n", src[i], dst[j]);
    }
    printf("end\n");
  }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    at = tmp_path_factory.mktemp("runs")
    (at / "runs.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "cuda-oxide-bench_b200" / "csrc"), str(at / "runs.cpp"),
                    "-o", str(at / "runs")], check=True)

    def run(lists):
        text = "\n".join(" ".join(map(str, [len(s), *s, *d])) for s, d in lists)
        out = subprocess.run([str(at / "runs")], input=text, capture_output=True, text=True, check=True).stdout
        return [[tuple(line.split()) for line in part.splitlines() if line] for part in out.split("end\n")[:-1]]

    return run


def planned(src, dst, P):
    """The plan of a copy as its description has it: -1 for what is left out."""
    sound = [(0 <= s < P and 0 <= d < P and s != d) for s, d in zip(src, dst)]
    sources = {s for s, ok in zip(src, sound) if ok}
    wanted = [d for d, ok in zip(dst, sound) if ok]
    return [d if ok and d not in sources and wanted.count(d) == 1 else -1 for d, ok in zip(dst, sound)]


def check(parts, lists):
    assert len(parts) == len(lists)
    for got, (src, dst) in zip(parts, lists):
        accepted = [(s, d) for s, d in zip(src, dst) if s >= 0 and d >= 0]
        # every accepted entry is written once, and nothing else
        assert sorted((int(x[1]), int(x[2])) for x in got if x[0] == "w") == sorted(accepted)
        # no source is read that no accepted entry has
        assert {int(x[1]) for x in got if x[0] == "r"} == {s for s, _ in accepted}


def test_sources_outside_the_pool_are_not_read(walk):
    P, far = 10, 2 ** 31 - 1
    lists = []
    for src, dst in [([10], [5]), ([far], [0]), ([far] * 9, list(range(9))), ([0, 1, 10, far, 2], [9, 8, 7, 6, 5]),
                     ([0, 1, 2, 3, 4, 10, 5, 6, 0], [9, 8, 8, 4, 7, 5, 99, 6, 3])]:
        lists.append((src, planned(src, dst, P)))
    check(walk(lists), lists)
    assert walk(lists)[:3] == [[], [], []]


def test_a_run_is_read_where_only_a_later_entry_stands(walk):
    """Forks of one page beyond the free ones, copies whose first destination is taken twice."""
    lists = [([3, 3, 3], [-1, 4, -1]), ([3] * 20, [-1] * 9 + [5] + [-1] * 10), ([3] * 8 + [4], [-1] * 8 + [1]),
             ([2, 2, -1, 2], [-1, -1, 6, 7])]
    check(walk(lists), lists)
    assert walk(lists)[0] == [("r", "3"), ("w", "3", "4")]


def test_random_lists(walk):
    rng = random.Random(5)
    lists = []
    for _ in range(300):
        P, n = rng.randrange(1, 30), rng.randrange(0, 40)
        src = []
        while len(src) < n:
            src += [rng.choice([-1, rng.randrange(P), P, P + 5, 2 ** 31 - 1])] * rng.randrange(1, 12)
        dst = [rng.randrange(-1, P + 1) for _ in range(n)]
        lists.append((src[:n], planned(src[:n], dst, P)))
    check(walk(lists), lists)
