"""CPU: the tiles that a block of windowed attention walks (csrc/window_walk.h), counted by a host
program against what each query sees: no tile more, none twice, none less; blocks behind a
sequence's end walk none."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "window_walk.h"

static long bad = 0, blocks = 0, padding = 0, whole = 0;

template <int TQ, int KT>
void block(int T, int n, int window, int sinks, int t0) {
  const dsa::Walk w = dsa::walk_of<TQ, KT>(n, window, sinks, t0);
  const int last = (t0 + TQ < n ? t0 + TQ : n) - 1;
  auto sees = [&](int t, int s) { return s <= t && (s > t - window || s < sinks); };
  // the steps that the kernel takes, in its three loops
  int steps = 0, v = 0, end = w.whole0 < w.total ? w.whole0 : w.total;
  for (; v < end; v += 2) steps += v + 1 < end ? 2 : 1;
  if (w.whole1 > w.whole0) {
    if (v != w.whole0 || (w.whole1 - w.whole0) % 2) ++bad;
    for (; v < w.whole1; v += 2, steps += 2)
      for (int i = v; i < v + 2; ++i, ++whole)
        for (int s = w.tile(i) * KT; s < w.tile(i) * KT + KT; ++s)
          for (int t = t0; t <= last; t += (t + 7 < last ? 7 : 1)) bad += !sees(t, s);
  }
  for (; v < w.total; v += 2) steps += v + 1 < w.total ? 2 : 1;
  int want = 0;
  for (int tile = 0; tile * KT <= last; ++tile) {
    bool any = false;
    for (int s = tile * KT; s < tile * KT + KT && !any; ++s) any = t0 <= last && s <= last && (s > t0 - window || s < sinks);
    int named = 0;
    for (int i = 0; i < w.total; ++i) named += w.tile(i) == tile;
    bad += named != (any ? 1 : 0);
    want += any;
  }
  if (steps != want || w.total != want) {
    if (bad < 5) printf("TQ=%d KT=%d T=%d n=%d window=%d sinks=%d t0=%d: %d steps, %d tiles\n", TQ, KT, T, n, window, sinks, t0, steps, want);
    ++bad;
  }
  ++blocks;
  padding += t0 >= n;
}

int main() {
  for (int T : {1, 64, 65, 130, 700})
    for (int n : {0, 1, 33, 64, 65, 127, 128, 129, 257, 448, 449, 640, 699, 700})
      for (int window : {1, 31, 64, 65, 100, 128, 129, 200, 449, 700})
        for (int sinks : {0, 1, 64, 70, 300, 700}) {
          if (n > T || window > T || sinks > T) continue;
          for (int t0 = 0; t0 < T; t0 += 64) {
            block<64, 64>(T, n, window, sinks, t0);
            block<64, 32>(T, n, window, sinks, t0);
            if (t0 % 128 == 0) block<128, 64>(T, n, window, sinks, t0);
          }
        }
  printf("%ld blocks, %ld behind the end, %ld whole tiles, %ld bad\n", blocks, padding, whole, bad);
  return bad || padding < 1000 || whole < 1000;
}
"""


def test_tiles_walked(tmp_path):
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    source, program = tmp_path / "walk.cpp", tmp_path / "walk"
    source.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(PKG, "csrc"), str(source), "-o", str(program)], check=True)
    r = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
