"""The order of waits on a shared-memory ring (csrc/yl_ring.h), run on the CPU.

Producer, copies, tensor-core thread and epilogue of the Newton-Schulz kernel
share a ring of three stages; a SQUARE tile has stages of its own that only the
epilogue reads and frees.  Barriers here have the hardware's meaning: a parity
wait passes when the phase of that parity is not the present one.  Copies land
in any order.  The tensor-core thread passes the epilogue's stages with the kernel's
own pass_stages and tells the epilogue, on two barriers in turn, what it has seen;
every product must find its own fill, whole, and no role may be left waiting."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "yumelayers_b200" / "csrc"

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "yl_ring.h"

constexpr int kStages = 3;
struct Barrier {
  unsigned phase = 0;
  bool passes(unsigned parity) const { return (phase & 1) != parity; }
};
struct Tile { int products, own; };

struct Ring {
  std::mt19937 rng;
  std::vector<Tile> tiles;
  Barrier full[kStages], empty[kStages];
  long content[kStages] = {-1, -1, -1};   // the fill that has landed, -1 while one is on its way
  std::vector<unsigned> flying;            // fills whose copies have not landed
  unsigned issued = 0, total = 0;
  std::vector<unsigned> epilogue;          // own stages in order
  std::vector<unsigned> tile_of;           // the tile whose sums the epilogue needs before that
  size_t ep = 0;
  std::vector<unsigned> square;            // and which of the tiles with own stages that is
  Barrier seen[2];
  unsigned handed = 0;                     // tiles whose last accumulator has been handed over
  bool free_unseen = false;
  bool bad = false;

  // One random move of another role; false when none of them can move.
  bool move() {
    const unsigned first = rng() % 3;
    for (unsigned k = 0; k < 3; ++k) {
      const unsigned who = (first + k) % 3;
      if (who == 0 && issued < total) {  // the producer issues a fill
        const unsigned s = issued % kStages;
        if (issued >= kStages && !empty[s].passes((issued / kStages - 1) & 1)) continue;
        content[s] = -1;
        flying.push_back(issued++);
        return true;
      }
      if (who == 1 && !flying.empty()) {  // some copy lands
        const size_t at = rng() % flying.size();
        const unsigned f = flying[at];
        flying.erase(flying.begin() + at);
        content[f % kStages] = f;
        ++full[f % kStages].phase;
        return true;
      }
      if (who == 2 && ep < epilogue.size() && handed > tile_of[ep]) {
        const unsigned f = epilogue[ep], j = square[ep];
        if (!free_unseen && !seen[j & 1].passes((j >> 1) & 1)) continue;
        if (!full[f % kStages].passes((f / kStages) & 1)) continue;
        if (content[f % kStages] != (long)f) bad = true;
        ++empty[f % kStages].phase;
        ++ep;
        return true;
      }
    }
    return false;
  }
};

int main(int argc, char** argv) {
  // 1: a walk that passes the epilogue's stages unseen, 2: an epilogue that does not wait
  // until they have been seen
  const int mistake = argc > 1 ? atoi(argv[1]) : 0;
  int wrong = 0;
  for (unsigned seed = 0; seed < 4000; ++seed) {
    Ring r;
    r.rng.seed(seed);
    r.free_unseen = mistake == 2;
    unsigned f = 0, squares = 0, walked = 0;
    for (int t = 0; t < 12; ++t) {
      const Tile tile{1 + (int)(r.rng() % 6), (int)(r.rng() % 3)};
      r.tiles.push_back(tile);
      f += tile.products;
      for (int e = 0; e < tile.own; ++e) {
        r.epilogue.push_back(f++);
        r.tile_of.push_back(t);
        r.square.push_back(squares);
      }
      squares += tile.own > 0;
    }
    r.total = f;
    uint32_t it = 0;
    auto landed = [&](uint32_t i) {
      for (unsigned k = r.rng() % 8; k; --k) r.move();
      while (!r.full[i % kStages].passes((i / kStages) & 1))
        if (!r.move()) return false;
      return true;
    };
    bool ok = true;
    for (const Tile& t : r.tiles) {
      for (int kb = 0; ok && kb < t.products; ++kb, ++it) {
        ok = landed(it);
        if (!ok) break;
        if (r.content[it % kStages] != (long)it) r.bad = true;
        ++r.empty[it % kStages].phase;
      }
      ++r.handed;
      if (mistake == 1) it += t.own;
      else ok = ok && yl::pass_stages(it, t.own, landed);
      if (ok && t.own > 0) ++r.seen[walked++ & 1].phase;
    }
    while (r.move()) {}
    if (!ok || r.bad || it != f || r.ep != r.epilogue.size()) ++wrong;
  }
  printf("%d\n", wrong);
}
"""


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "model.cpp").write_text(MODEL)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{CSRC}", str(d / "model.cpp"), "-o",
                    str(d / "model")], check=True)
    return lambda *a: int(subprocess.run([d / "model", *a], check=True, capture_output=True,
                                         text=True, timeout=120).stdout)


def test_every_product_finds_its_own_fill(model):
    assert model() == 0


def test_the_model_sees_a_stage_that_is_not_waited_for(model):
    """The same walk past the epilogue's stages without their waits."""
    assert model("1") > 0


def test_the_model_sees_a_stage_freed_too_early(model):
    """The epilogue frees a stage, and the producer fills it again, before the walk has
    seen it: the walk waits for a phase that has gone by."""
    assert model("2") > 0
