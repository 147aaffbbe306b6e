"""CPU: the turns of the attention gradients' row tiles on two operand buffers (csrc/row_turns.cuh), stepped against a model of the barriers under random interleavings.

Three parties meet each row tile in turn: copies in, elements (which put the results into the operand buffer) and copies out, the last with other work of any length between two tiles.  A barrier
is waited for by parity, so two phases that complete before the waiter looks are none to it.  One "staged" barrier for both buffers (a planted mistake) must be caught by the model."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "row_turns.cuh"

struct Barrier {
  uint32_t done = 0;                                                      // phases completed
  bool passed(uint32_t parity) const { return (done & 1u) != parity; }    // try_wait.parity
};
enum { FREE, LOADED, STAGED };

// 0: every row tile was loaded, staged and copied out once, in order; 1: a buffer was used by the wrong tile; 2: a wait that never ends
int run(uint32_t tiles, uint32_t most_work, uint32_t seed, bool planted) {
  std::mt19937 rng(seed);
  Barrier full[2], empty[2], staged[2];
  int state[2] = {FREE, FREE};
  uint32_t tile[2] = {0, 0};
  fovi::RowTurn in, elements, out;
  uint32_t work = 0;                                                      // of the copying warp, before it looks for the next tile
  for (uint64_t spin = 0; out.seq < tiles && spin < 100ull * tiles * (most_work + 10); ++spin) {
    switch (rng() % 3) {
      case 0: {
        if (in.seq >= tiles || !empty[in.buffer()].passed(in.parity() ^ 1u)) break;
        const uint32_t f = in.buffer();
        if (state[f] != FREE) return 1;
        state[f] = LOADED; tile[f] = in.seq; ++full[f].done;
        in.next();
        break;
      }
      case 1: {
        if (elements.seq >= tiles || !full[elements.buffer()].passed(elements.parity())) break;
        const uint32_t f = elements.buffer();
        if (state[f] != LOADED || tile[f] != elements.seq) return 1;
        state[f] = STAGED; ++staged[planted ? 0 : f].done;
        elements.next();
        break;
      }
      default: {
        if (work) { --work; break; }
        const uint32_t f = out.buffer();
        if (!(planted ? staged[0].passed(out.seq & 1u) : staged[f].passed(out.parity()))) break;
        if (state[f] != STAGED || tile[f] != out.seq) return 1;
        state[f] = FREE; ++empty[f].done;
        out.next();
        work = most_work ? rng() % most_work : 0;
      }
    }
  }
  return out.seq == tiles ? 0 : 2;
}

int main(int argc, char** argv) {
  int seen = 0;
  for (uint32_t seed = 0; seed < 200; ++seed) seen |= 1 << run(60, (uint32_t)atoi(argv[1]), seed, atoi(argv[2]) != 0);
  printf("%d\n", seen);
  return 0;
}
"""


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    d = tmp_path_factory.mktemp("turns")
    src, exe = d / "model.cpp", d / "model"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "fovi_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    return lambda work, planted: int(subprocess.run([str(exe), str(work), str(int(planted))], check=True, capture_output=True, text=True).stdout)


@pytest.mark.parametrize("work", (0, 1, 5, 50, 300))
def test_every_row_tile_is_staged_and_copied_out(model, work):
    assert model(work, False) == 1 << 0


@pytest.mark.parametrize("work", (5, 50))
def test_the_model_catches_one_barrier_for_both_buffers(model, work):
    assert model(work, True) & (1 << 2)


def test_the_kernel_takes_these_turns():
    """Each of the three barriers is there once for each buffer, and the kernel waits for it with the turn's own buffer and parity."""
    with open(os.path.join(ROOT, "fovi_b200", "csrc", "attention_tc_grad.cu")) as f:
        text = f.read()
    for name, turn in (("row_empty", "fp ^ 1u"), ("row_full", "w.row.parity()"), ("staged", "w.row.parity()")):
        assert f"{name}[2]" in text
        assert f"hdr->{name}[f]), {turn}," in text, name
    assert "const uint32_t f = w.row.buffer(), fp = w.row.parity()" in text and "hdr->staged[turn.buffer()]" in text
