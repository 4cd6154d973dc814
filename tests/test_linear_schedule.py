"""The schedule of the CTA pairs' kernel (csrc/kernels/linear_schedule.h, the code that the kernel itself runs), compiled for the
host: every 256 x 128 piece of each output belongs to exactly one tile of one pair."""

import os
import shutil
import subprocess

import pytest

from torch_vulkan_b200 import _build

MAIN = r"""
#include <cstdio>
#include <cstdlib>
#include "linear_schedule.h"
using namespace tvb;

static PairExtent extent(int halves, int j, int i, int blocks) {
  PairExtent e{};
  if (j == 0 || i == 0) return e;
  e.I = i; e.J = j; e.blocks = blocks;
  e.tiles_i = (i + kTileI - 1) / kTileI;
  e.tiles_j = (j + halves * kHalfJ - 1) / (halves * kHalfJ);
  e.tiles = e.tiles_i * e.tiles_j;
  return e;
}

template <int HALVES>
static int run(char** v) {
  const PairExtent e0 = extent(HALVES, atoi(v[0]), atoi(v[1]), atoi(v[2])), e1 = extent(HALVES, atoi(v[3]), atoi(v[4]), atoi(v[5]));
  PairPlan plan;
  const int pairs = plan_pairs<HALVES>(e0, e1, atoi(v[6]), &plan);
  std::printf("pairs %d cut %d whole %d extra %d\n", pairs, plan.cut_cols, plan.whole, plan.extra);
  for (int pair = 0; pair < pairs; pair++) {
    PairSchedule<HALVES> s(plan, e0, pair, pairs);
    PairTile t;
    while (s.next(plan, e0, e1, t)) std::printf("%d %d %d %d %d %d\n", pair, t.product, t.row, t.col, t.cols, t.halves);
  }
  return 0;
}

int main(int argc, char** v) { return argc != 9 ? 2 : v[1][0] == '2' ? run<2>(v + 2) : run<1>(v + 2); }
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no g++ here")
    folder = tmp_path_factory.mktemp("schedule")
    (folder / "main.cpp").write_text(MAIN)
    out = str(folder / "schedule")
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(_build.CSRC, "kernels"), str(folder / "main.cpp"), "-o", out], check=True)
    return out


def tiles_of(program, halves, first, second, pairs):
    done = subprocess.run([program, *map(str, (halves, *first, *second, pairs))], capture_output=True, text=True, check=True)
    lines = done.stdout.splitlines()
    head = lines[0].split()
    return {head[i]: int(head[i + 1]) for i in range(0, len(head), 2)}, [tuple(map(int, line.split())) for line in lines[1:]]


# (rows, columns, steps of r) of the two products (the first with the longer r, or empty), pairs that run at once
TWO = [((2048, 4096, 224), (14336, 4096, 32), 74), ((300, 600, 100), (5000, 1100, 7), 74), ((1000, 1000, 16), (1000, 1024, 16), 74),
       ((513, 257, 3), (511, 255, 2), 2), ((9000, 900, 9), (700, 9000, 9), 74), ((2049, 2049, 33), (8200, 2100, 32), 74),
       ((4100, 1800, 29), (1900, 4100, 29), 74), ((257, 256, 1000000), (66000, 4096, 1), 74), ((2560, 2560, 7), (2560, 2304, 5), 67),
       ((256, 256, 5), (256, 256, 5), 74)]
ONE = [((0, 0, 0), (2048, 14336, 64), 74), ((0, 0, 0), (257, 300, 5), 74), ((0, 0, 0), (66000, 36000, 1), 74), ((0, 0, 0), (1900, 2603, 128), 74),
       ((0, 0, 0), (2100, 2600, 129), 74), ((0, 0, 0), (65, 18944, 10), 74), ((0, 0, 0), (4863, 4865, 200), 74), ((0, 0, 0), (1, 1, 1), 74),
       ((0, 0, 0), (512, 256 * 75, 9), 74), ((0, 0, 0), (2049, 2817, 9), 71)]


@pytest.mark.parametrize("halves,first,second,pairs", [(1, *c) for c in TWO + ONE] + [(2, *c) for c in ONE])
def test_every_piece_of_the_outputs_is_one_pairs(program, halves, first, second, pairs):
    plan, tiles = tiles_of(program, halves, first, second, pairs)
    assert 1 <= plan["pairs"] <= pairs and plan["cut"] in (128, 256)
    seen, order = set(), {}
    for pair, product, row, col, cols, parts in tiles:
        assert 0 <= pair < plan["pairs"] and parts in ((1, 2) if halves == 2 else (1,)) and cols in (256, plan["cut"])
        rows, columns = (first, second)[product][:2]
        assert row % 256 == 0 and col % 128 == 0 and row < rows and col < columns  # (a store never begins outside)
        assert row + 256 * (parts - 1) < rows
        assert order.setdefault(pair, 0) <= product  # (a pair goes from product 0 to product 1 once)
        order[pair] = product
        for r in range(row, row + 256 * parts, 256):
            for c in range(col, col + cols, 128):
                assert (product, r, c) not in seen
                seen.add((product, r, c))
    want = sum(-(-j // 256) * -(-i // 128) for j, i, _ in (first, second))
    inside = sum(1 for product, r, c in seen if r < (first, second)[product][0] and c < (first, second)[product][1])
    assert inside == want
    # no pair is left without work while another has more than a tile of the same product to spare
    if first[0] == 0:
        load = [0] * plan["pairs"]
        for pair, _, _, _, cols, parts in tiles:
            load[pair] += parts * cols
        assert max(load) - min(load) <= 256 * halves
