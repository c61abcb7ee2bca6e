// Index arithmetic of the paged key / value cache, shared by its kernels and, as plain C++, by a host test.
//
// The device arrays that a call brings (lengths, row starts, page numbers) are not checked on the host, which would
// wait for them; everything read from them is brought into range here instead, so that no value in them makes a
// kernel read or write outside the call's buffers or loop without end.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define TARS_HD __host__ __device__ __forceinline__
#else
#define TARS_HD inline
#endif

namespace tars {

TARS_HD int imin(int a, int b) { return a < b ? a : b; }
TARS_HD int imax(int a, int b) { return a > b ? a : b; }
TARS_HD int iclamp(int x, int lo, int hi) { return imin(imax(x, lo), hi); }
TARS_HD int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Positions that sequence b's cache holds: lens[b] within what its table row can name (cap, at most 2^30).
TARS_HD int seq_len(const int32_t* lens, int b, int cap) { return iclamp(lens[b], 0, cap); }

// Rows [first, first + n) of sequence b among `rows` packed rows.
struct RowSpan {
  int first, n;
};
TARS_HD RowSpan seq_rows(const int32_t* starts, int b, int rows) {
  const int r0 = iclamp(starts[b], 0, rows);
  return {r0, imax(iclamp(starts[b + 1], 0, rows) - r0, 0)};
}

// Tiles of m rows over the packed rows, each row `group` deep, none with rows of two sequences: those of sequence b are
// numbered from tile_first(b) on. A closed form, in place of a sum over the sequences before: floor(s group / m) + b
// leaves ceil(n group / m) numbers or one more to a sequence of n rows.
TARS_HD int tile_first(const int32_t* starts, int b, int rows, int group, int m) {
  return iclamp(starts[b], 0, rows) * group / m + b;
}

// Of n rows' ceil(n group / m) tiles, rows at positions p0 .. p0 + n - 1: how many, the last ones, have their last row
// behind the first s - 1 steps of `step` positions; all of them for s <= 0.
TARS_HD int tiles_behind(int s, int p0, int n, int group, int m, int step) {
  const int tiles = ceil_div(n * group, m);
  if (s <= 0) return tiles;
  const int token = imax((s - 1) * step - p0, 0);  // the first row that is
  return token < n ? tiles - (ceil_div(token * group + 1, m) - 1) : 0;
}

// Whether the row at position p sees position j >= 0: not ahead of it, and within the window (0: none) or a first token.
TARS_HD bool sees(int p, int j, int window, int sinks) {
  return j <= p && (window == 0 || j > p - window || j < sinks);
}

// Of the columns [c0, c0 + cols), `group` of them to a row, rows at positions p0, p0 + 1, ...: the ones that see position j >= 0
// are c0 + lo .. c0 + hi - 1 (lo >= hi: none).
struct Range {
  int lo, hi;
};
TARS_HD Range seen_by(int j, int p0, int group, int c0, int cols, int window, int sinks) {
  const int rows = ceil_div(c0 + cols, group);  // no row behind them counts
  const int64_t after = window == 0 || j < sinks ? rows : int64_t{j} - p0 + window;
  const int first = iclamp(j - p0, 0, rows), end = after < 0 ? 0 : after > rows ? rows : static_cast<int>(after);
  return {iclamp(first * group - c0, 0, cols), iclamp(end * group - c0, 0, cols)};
}

// The steps of `step` positions that hold every position seen by a row at a position in [plo, phi] of a sequence of
// length len: [0, a) and [b0, b1), a <= b0 <= b1. A step of the first part may hold positions of the window, and
// steps of either may hold positions that a row does not see.
struct Steps {
  int a, b0, b1;
  TARS_HD int n() const { return a + b1 - b0; }
  TARS_HD int at(int i) const { return i < a ? i : i - a + b0; }
};
TARS_HD Steps visible_steps(int plo, int phi, int len, int window, int sinks, int step) {
  const int end = imax(imin(phi + 1, len), 0);
  const int b1 = ceil_div(end, step);
  const int lo = window == 0 ? 0 : imax(imax(plo, 0) - window + 1, 0);
  const int a = imin(ceil_div(imin(sinks, lo), step), b1);
  return {a, imin(imax(lo / step, a), b1), b1};
}

}  // namespace tars
