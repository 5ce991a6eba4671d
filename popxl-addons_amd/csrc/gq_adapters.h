// Low-rank adapters: the plan of a batch, shared by the kernels that make and read it.
#pragma once
#include "gq_common.h"

namespace gq {

constexpr int kAdapterSmallTile = 16, kAdapterLargeTile = 64;  // rows of one adapter that a workgroup takes together
constexpr int kAdapterSegment = 2048;                          // rows that one part of a weight gradient sums over
constexpr int kMostAdapters = 2048;

struct AdapterTile {
  int adapter;  // -1: rows without one
  int begin, count;
  int first;  // segments: where its tiles begin in the list of small ones (small tiles) and of large ones, and
  int first_large, part, spare;  // the part it writes, -1 where it is its adapter's only one
};

// Where the arrays of a plan lie (4-byte words from its start).  Sizes depend on the numbers of rows and adapters alone;
// the counts (how many tiles there are) are device data.
struct PlanLayout {
  int64_t rows, adapters;
  int64_t counts, order, parts, small, large, segments, words;
  int64_t most_small, most_large, most_segments, most_parts;
  PlanLayout(int64_t rows_, int64_t adapters_) : rows(rows_), adapters(adapters_) {
    const int64_t kinds = rows < adapters + 1 ? rows : adapters + 1;
    most_small = rows / kAdapterSmallTile + kinds, most_large = rows / kAdapterLargeTile + kinds;
    most_segments = rows / kAdapterSegment + kinds;
    most_parts = 2 * rows / kAdapterSegment;  // an adapter of s >= 2 segments has more than 2048 (s - 1) >= 1024 s rows
    int64_t at = 0;
    const auto take = [&](int64_t n) {
      const int64_t here = at;
      at += (n + 63) / 64 * 64;
      return here;
    };
    counts = take(64);               // small tiles, large tiles, segments, parts
    order = take(rows);              // the rows, by adapter and then by index; those without one last
    parts = take(2 * adapters);      // of each adapter: its first part, its segments
    small = take(8 * most_small), large = take(8 * most_large), segments = take(8 * most_segments);
    words = at;
  }
};

}  // namespace gq
