// Which rows of a call's tensors share places in memory, from their strides (host only). A
// kernel's workgroups write rows in any order, beside others that still read.
#ifndef CUDALM_ROW_PLACES_H
#define CUDALM_ROW_PLACES_H

#include <stdint.h>

namespace cudalm_hip {

// `count` rows, `step` 16-bit elements apart, of `side` pieces each, `between` apart, of
// `width` elements. Strides of either sign.
struct RowGrid {
  const void* at;
  int64_t count, step, side, between, width;
};

typedef __int128 place_t;  // products of any counts and strides

// Whether lo < c + s step < hi for some whole s, |s| < n.
inline bool steps_meet(place_t c, place_t n, place_t step, place_t lo, place_t hi) {
  if (n < 2 || step == 0) return lo < c && c < hi;
  if (step < 0) step = -step;
  const place_t a = lo - c;
  place_t s = a / step - (a % step < 0 ? 1 : 0) + 1;  // the first one past lo
  if (s < 1 - n) s = 1 - n;
  return s < n && c + s * step < hi;
}

// Whether no two pieces share an element. (Where rows lie one after the other, or pieces' columns
// do, that is seen at once; other layouts are gone through.)
inline bool places_apart(const RowGrid& g) {
  place_t n = g.count, step = g.step < 0 ? -static_cast<place_t>(g.step) : g.step;
  place_t m = g.side, between = g.between < 0 ? -static_cast<place_t>(g.between) : g.between;
  if (n < 1 || m < 1) return true;
  if ((n > 1 && step < g.width) || (m > 1 && between < g.width)) return false;
  if (n < 2 || m < 2 || step >= (m - 1) * between + g.width || between >= (n - 1) * step + g.width) return true;
  if (m > n) {
    place_t t = n;
    n = m, m = t, t = step, step = between, between = t;
  }
  for (place_t t = 1; t < m; ++t)
    if (steps_meet(t * between, n, step, -static_cast<place_t>(g.width), g.width)) return false;
  return true;
}

// Whether pieces of a and b share an element. Of grids whose strides differ this is not found
// out (false), unless there is one row of each.
inline bool places_meet(const RowGrid& a, const RowGrid& b) {
  if (a.count != b.count || a.count < 1 || a.side < 1 || b.side < 1) return false;
  const place_t n = a.count, between = a.side > 1 ? a.between : b.side > 1 ? b.between : 0;
  const place_t step = n > 1 ? a.step : 0;
  if ((n > 1 && a.step != b.step) || (a.side > 1 && b.side > 1 && a.between != b.between)) return false;
  const place_t d = (static_cast<place_t>(reinterpret_cast<uintptr_t>(b.at)) -
                     static_cast<place_t>(reinterpret_cast<uintptr_t>(a.at))) / 2;
  // both as a whole, which is all there is to tensors of their own; then whole rows; then pieces
  const place_t length = (n - 1) * (step < 0 ? -step : step);
  const place_t low_a = between < 0 ? (a.side - 1) * between : 0, low_b = between < 0 ? (b.side - 1) * between : 0;
  const place_t span_a = (a.side - 1) * (between < 0 ? -between : between) + a.width;
  const place_t span_b = (b.side - 1) * (between < 0 ? -between : between) + b.width;
  const place_t rows = d + low_b - low_a;
  if (rows - length >= span_a || rows + length <= -span_b) return false;
  if (!steps_meet(rows, n, step, -span_b, span_a)) return false;
  for (place_t t = 1 - a.side; t < b.side; ++t)
    if (steps_meet(d + t * between, n, step, -static_cast<place_t>(b.width), a.width)) return true;
  return false;
}

}  // namespace cudalm_hip

#endif
