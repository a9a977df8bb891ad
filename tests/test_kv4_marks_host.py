"""The marks of columns without numbers (kv4_marks.h), run by two waves one of which is always late: it goes on after a
barrier only when the other waits at the next one.  Host code; no GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from karume_amd import build

SHIM = """
#include <condition_variable>
#include <cstring>
#include <mutex>
#include <thread>
#include "kv4_marks.h"

// Two threads of which one runs at a time; barriers are told by their place, and both have to come to the same ones.
struct Turns {
  std::mutex m;
  std::condition_variable cv;
  int running, fast, place[2] = {-1, -1};
  bool ended[2] = {false, false}, apart = false;

  void hand_to(std::unique_lock<std::mutex>& lock, int to, int me) {
    running = to;
    cv.notify_all();
    cv.wait(lock, [&] { return running == me; });
  }
  void barrier(int me, int at) {
    std::unique_lock<std::mutex> lock(m);
    place[me] = at;
    if (ended[1 - me]) {   // no one to wait for: a barrier more than the other has
      apart = true;
      return;
    }
    if (me != fast && place[0] != place[1]) apart = true;   // (the fast one has arrived before it)
    hand_to(lock, 1 - me, me);
  }
  void end(int me) {
    std::unique_lock<std::mutex> lock(m);
    ended[me] = true;
    running = 1 - me;
    cv.notify_all();
  }
};

constexpr int kColumns = 8;
// Tiles of a piece as kv4_chunk_kernel takes them: wave 0 makes values, and so marks, before it multiplies, wave 1 has no
// part in the marks but reads them.  mark[tile]: groups of the tile's column tile % kColumns.
extern "C" int piece(int tiles, const uint32_t* mark, int fast, int* wrong) {
  static krm::Kv4Marks<kColumns> marks;
  memset(&marks, 0xff, sizeof marks);
  Turns turns;
  turns.running = turns.fast = fast;
  int bad[2] = {0, 0};
  auto wave = [&](int me) {
    {
      std::unique_lock<std::mutex> lock(turns.m);
      turns.cv.wait(lock, [&] { return turns.running == me; });
    }
    int at = 0;
    marks.clear(me, 2);
    turns.barrier(me, at++);
    for (int tile = -1; tile < tiles; ++tile) {
      const uint32_t buffer = (uint32_t)tile & 1u, other = buffer ^ 1u;
      if (me == 0 && tile + 1 < tiles && mark[tile + 1]) {
        marks.groups[other][(tile + 1) % kColumns] |= mark[tile + 1];
        marks.any[other] = 1;
      }
      if (tile >= 0) {
        bad[me] += (marks.any[buffer] != 0) != (mark[tile] != 0);
        for (int i = 0; i < kColumns; ++i)
          bad[me] += marks.groups[buffer][i] != (i == tile % kColumns ? mark[tile] : 0u);
      }
      marks.end_turn(buffer, me, 2, [&] { turns.barrier(me, at++); });
    }
    turns.end(me);
  };
  std::thread first(wave, 0), second(wave, 1);
  first.join();
  second.join();
  *wrong = bad[0] + bad[1];
  return turns.apart;
}
"""


@pytest.fixture(scope="module")
def piece(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no compiler")
    at = tmp_path_factory.mktemp("marks")
    (at / "shim.cpp").write_text(SHIM)
    library = os.path.join(at, "shim.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-pthread", "-shared", "-fPIC", "-I", build.CSRC,
                    str(at / "shim.cpp"), "-o", library], check=True)

    def run(marks, fast):
        wrong = C.c_int(-1)
        apart = C.CDLL(library).piece(len(marks), (C.c_uint32 * len(marks))(*marks), fast, C.byref(wrong))
        return apart, wrong.value
    return run


@pytest.mark.parametrize("fast", [0, 1])
@pytest.mark.parametrize("pattern", range(64))
def test_a_late_wave_takes_the_same_barriers_and_sees_the_same_marks(piece, fast, pattern):
    """Every order of marked tiles and others, one after the other and two tiles (one buffer) apart."""
    marks = [(3 + tile if pattern >> tile & 1 else 0) for tile in range(6)]
    assert piece(marks, fast) == (0, 0)
