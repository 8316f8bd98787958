"""The kernels' own index arithmetic (csrc/index.h), built for the host: pages of units, orders of tiles, LDS slots, groups of scales."""
import ctypes as C
import random
import subprocess

import pytest

from sparsefold_amd import _build

SHIM = """
#include "index.h"
extern "C" {
int page(uint32_t unit, uint32_t per) { return page_of(page_div(per), unit); }
void banded(int band, int t, int gx, int gy, int* at) {
  if (band == 5) banded_tile<5>(t, gx, gy, at[0], at[1]);
  else banded_tile<8>(t, gx, gy, at[0], at[1]);
}
int on_xcd(int b, int total) { return tile_on_xcd(b, total); }
void walk(int b, int total, int* at) {
  const TileWalk w = tiles_on_xcd(b, total);
  at[0] = w.first;
  at[1] = w.end;
}
int slot(int eight, int row, int piece) { return eight ? tile_slot<true>(row, piece) : tile_slot<false>(row, piece); }
int group(int g, int blocks) { return scales_of_group(g, blocks); }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
  at = tmp_path_factory.mktemp("index")
  (at / "shim.hip").write_text(SHIM)
  subprocess.run([_build.hipcc(), "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-shared", f"-I{_build.CSRC}", str(at / "shim.hip"), "-o", str(at / "shim.so")],
                 check=True, capture_output=True, text=True)
  return C.CDLL(str(at / "shim.so"))


def pair(f, *args):
  at = (C.c_int * 2)()
  f(*args, at)
  return at[0], at[1]


@pytest.mark.parametrize("per", [1, 2, 3, 4, 5, 7, 8, 12, 63, 64, 65, 100, 1000, 4095, 1 << 20, (1 << 26) - 1, 1 << 26])
def test_page_of_a_unit(index, per):
  rng = random.Random(per)
  edge = [k * per + d for k in (0, 1, 2, 3, 17, (1 << 27) // per - 1, (1 << 27) // per) for d in (-1, 0, 1)]
  for unit in edge + [rng.randrange(1 << 27) for _ in range(2000)]:
    if 0 <= unit < 1 << 27:
      assert index.page(unit, per) == unit // per


GRIDS = [(1, 1), (1, 1025), (1030, 1), (9, 131), (40, 32), (63, 64), (129, 8), (33, 33), (7, 300), (4, 40), (16, 10), (17, 17), (32, 32), (5, 33)]


@pytest.mark.parametrize("band", [5, 8])
@pytest.mark.parametrize("gx,gy", GRIDS)
def test_bands_hold_every_tile_once(index, gx, gy, band):
  seen = [pair(index.banded, band, t, gx, gy) for t in range(gx * gy)]
  assert set(seen) == {(x, y) for x in range(gx) for y in range(gy)}
  assert [x // band for x, _ in seen] == sorted(x // band for x, _ in seen)


@pytest.mark.parametrize("total", [1, 7, 8, 9, 63, 160, 1025, 1179, 4032])
def test_each_tile_has_one_workgroup(index, total):
  """One workgroup a tile: contiguous ranges, XCD by XCD."""
  order = [index.on_xcd(b, total) for b in range(total)]
  assert sorted(order) == list(range(total))
  for xcd in range(8):
    mine = order[xcd::8]
    assert mine == list(range(mine[0], mine[0] + len(mine))) if mine else True


@pytest.mark.parametrize("total", [160, 161, 167, 168, 255, 256, 257, 289, 1000, 1024, 5000])
@pytest.mark.parametrize("resident", [8, 32, 256, 512])
def test_walks_reach_each_tile_once(index, total, resident):
  """Persistent workgroups, at most as many as tiles in whole eights."""
  workgroups, seen = min(resident, (total + 7) // 8 * 8), []
  for b in range(workgroups):
    t, end = pair(index.walk, b, total)
    while t < end:
      seen.append(t)
      t += workgroups // 8
  assert sorted(seen) == list(range(total))


@pytest.mark.parametrize("eight", [0, 1])
def test_slots_are_a_permutation(index, eight):
  """A row's pieces lie on all of its slots; 16 rows read together (one piece each) on 16 different ones of 256 bytes."""
  pieces = 8 if eight else 4
  for r in range(128):
    assert {index.slot(eight, r, p) for p in range(pieces)} == set(range(pieces))
  for r0 in range(0, 128, 16):
    for p in range(pieces):
      assert len({(r * pieces * 16 + index.slot(eight, r, p) * 16) % 256 for r in range(r0, r0 + 16)}) == 16


@pytest.mark.parametrize("K", range(512, 5000, 128))
@pytest.mark.parametrize("per_step", [2, 4])
def test_groups_of_scales_stay_in_their_rows(index, K, per_step):
  """16 scales a group, inside the row and at a whole word; a step's scales lie in its group's, at a whole word but for the half word of a
  64-k step."""
  blocks, steps = K // 32, 16 // per_step
  for t in range(K // (32 * per_step)):
    first = index.group(t // steps, blocks)
    assert 0 <= first <= blocks - 16 and first % 4 == 0
    at = per_step * t - first
    assert 0 <= at and at + per_step <= 16 and (at % 4 == 0 or per_step == 2)
