"""Whether two strided views share an element (csrc/nk_views.h, host code) against every element of both, compiled by itself."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include "nk_views.h"
#include <cstdio>
int main() {
    int tries;
    for (nk::View v[2]; scanf("%d", &tries) == 1;) {
        for (auto& x : v) {
            long long first, extent, step;
            if (scanf("%lld %d", &first, &x.rank) != 2) return 1;
            x.first = first;
            for (int k = 0; k < x.rank; k++) {
                if (scanf("%lld %lld", &extent, &step) != 2) return 1;
                x.extent[k] = extent; x.step[k] = step;
            }
        }
        printf("%d\n", (int)nk::views_meet(v[0], v[1], tries));
    }
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    at = tmp_path_factory.mktemp("views")
    (at / "views.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-O1", "-I", os.path.join(ROOT, "neureka_amd", "csrc"), str(at / "views.cpp"), "-o", str(at / "views")], check=True)

    def answers(cases, tries=20000):
        text = "\n".join(" ".join(map(str, [tries] + [n for first, axes in pair for n in [first, len(axes)] + [m for a in axes for m in a]])) for pair in cases)
        out = subprocess.run([str(at / "views")], input=text, capture_output=True, text=True, check=True, timeout=60).stdout
        return [bool(int(line)) for line in out.split()]
    return answers


def elements(view):
    found = {view[0]}
    for extent, step in view[1]:
        found = {a + step * i for a in found for i in range(extent)}
    return found


def test_against_all_elements(meet):
    rng = random.Random(1)
    cases = []
    for _ in range(4000):
        pair = []
        for _ in range(2):
            pair.append((rng.randrange(-40, 40), [(rng.randrange(1, 6), rng.choice((0, 1, 1, 2, 3, 5, 7, 10, 12, 30, -1, -6))) for _ in range(rng.randrange(0, 5))]))
        cases.append(tuple(pair))
    want = [bool(elements(a) & elements(b)) for a, b in cases]
    assert 0.2 < sum(want) / len(want) < 0.9
    assert meet(cases) == want


def test_views_of_large_matrices(meet):
    rows = (0, [(30000, 60000), (30000, 1)])                                  # the left half of a matrix of 30000 x 60000 ...
    cases = [(rows, (30000, [(30000, 60000), (30000, 1)])),                   # ... against its right half
             (rows, (29999, [(30000, 60000), (30000, 1)])),                   # ... one column earlier
             ((0, [(20000, 40000), (20000, 2)]), (1, [(20000, 40000), (20000, 2)])),      # even and odd columns
             ((0, [(20000, 40000), (20000, 2)]), (40000, [(20000, 80000), (5, 2)])),
             ((0, [(40000, 40000), (40000, 1)]), (0, [(40000, 1), (40000, 40000)])),      # a matrix and its transpose
             ((0, [(100, 40000), (100, 1)]), (100, [(100, 1), (100, 40000)])),            # a square and the transpose of its right neighbour
             ((0, [(7, 1)]), (7, [(7, 1)])), ((0, [(8, 1)]), (7, [(7, 1)]))]
    assert meet(cases) == [False, True, False, True, True, False, False, True]


def test_a_search_that_gives_up_says_yes(meet):
    pair = ((0, [(5, 1000), (5, 100)]), (60, [(3, 10)]))
    assert meet([pair]) == [False] and meet([pair], tries=0) == [True]
