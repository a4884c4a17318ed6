"""How the products of the head's loss are tiled and split (``csrc/head_plan.hpp``, compiled for the host with g++): the
calls that the GPU tests make for the sake of a path do take it."""
import shutil
import subprocess
from pathlib import Path

import pytest

from lm_paths import HEAD_PATHS

CSRC = Path(__file__).resolve().parent.parent / "monarch_muon_amd" / "csrc"

PROG = r'''
#include <stdio.h>
#include "head_plan.hpp"
using namespace mmuon;
static void show(const HeadPlan& p, int64_t m, int64_t n, const char* end) {
  printf("%d %s%s", p.cols(), p.full >= p.tiles(m, n) ? "whole" : p.full == 0 ? "all" : "tail", end);
}
int main() {
  long long t, d, v, train;
  while (scanf("%lld %lld %lld %lld", &t, &d, &v, &train) == 4) {
    const HeadPlans p = head_plans(t, d, v, train != 0);
    show(p.logits, v, t, ", ");
    show(p.dx, d, t, ", ");
    show(p.dw, d, v, "\n");
  }
  return 0;
}
'''


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = (tmp_path_factory.mktemp("plan") / n for n in ("p.cpp", "p"))
    src.write_text(PROG)
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)

    def run(*calls):
        text = "".join(" ".join(map(str, c)) + "\n" for c in calls)
        return subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
    return run


def test_paths_are_what_their_rows_say(plans):
    calls = [(piece or T, D, V, 1) for (T, D, V, piece), _ in HEAD_PATHS]
    assert plans(*calls) == [path for _, path in HEAD_PATHS]


def test_paths_cover_every_tiling(plans):
    """Every tile and split that a product takes is among the rows, the logits' splits in pieces too."""
    for product, kinds in enumerate((["128 whole", "128 tail", "128 all", "256 whole", "256 tail", "256 all"],
                                     ["128 whole", "128 tail", "128 all", "256 whole", "256 tail", "256 all"],
                                     ["256 whole", "256 tail", "256 all"])):
        assert set(kinds) == {path.split(", ")[product] for _, path in HEAD_PATHS}


def test_loss_alone_of_few_tokens_is_in_small_tiles(plans):
    assert [p.split(",")[0] for p in plans((1, 4096, 50304, 0), (64, 512, 50257, 0), (65, 512, 50257, 0),
                                           (64, 512, 50257, 1))] == ["64 whole", "64 whole", "128 whole", "128 whole"]
