// window_walk.h -- which tiles of keys a block of queries of dsa_window_attention walks.  Integers
// alone, so that host code can count them too (constexpr: callable from both).
#pragma once

namespace dsa {

// Tiles of KT keys for the TQ queries from t0 on, of a sequence of n tokens: those of the first
// tokens, 0 .. first - 1, then near, near + 1, ... up to the last query's own; the walk's steps are
// 0 .. total - 1.  None where all queries are behind the sequence's end.
struct Walk {
  int n;
  int first, near;
  int total;
  int whole0, whole1;  // steps of tiles that all queries see whole: even numbers, for two buffers in turn

  constexpr int tile(int step) const { return step < first ? step : near + step - first; }
};

constexpr int at_most(int a, int b) { return a < b ? a : b; }
constexpr int at_least(int a, int b) { return a > b ? a : b; }

template <int TQ, int KT>
constexpr Walk walk_of(int n, int window, int sinks, int t0) {
  Walk w{n, 0, 0, 0, 0, 0};
  if (t0 >= n) return w;
  const int last = at_most(t0 + TQ, n) - 1;
  w.near = at_least(0, t0 - window + 1) / KT;
  w.first = at_most((sinks + KT - 1) / KT, w.near);
  w.total = w.first + last / KT - w.near + 1;
  // from the first tile that the last query sees whole to the last one before all queries
  const int seen = last >= window ? (last - window) / KT + 1 : 0;
  w.whole0 = (w.first + at_least(0, seen - w.near) + 1) & ~1;
  w.whole1 = w.whole0 + at_least(0, (w.first + t0 / KT - w.near - w.whole0) & ~1);
  return w;
}

}  // namespace dsa
