// Where the join of attention with shared prefixes finds a segment's parts.
#ifndef CUDALM_PAGED_PLACES_H
#define CUDALM_PAGED_PLACES_H

namespace cudalm_hip {

// Part y of a segment's own tokens is at first, first + 1, first + 3, ..; its prefix has parts
// 0 .. prefix - 1, with the sequence's first row at `row`.
struct SegmentParts {
  int first, own, prefix, row;
};

constexpr int own_part(int first, int y) { return first + (y ? 2 * y - 1 : 0); }

constexpr int within(int x, int lo, int hi) { return x < lo ? lo : x < hi ? x : hi; }

// What a segment's entry says, and nothing past `slots` own parts, `splits` parts of a prefix and
// prefix_rows - rows rows: where lengths change under the call an entry may not have been written.
constexpr SegmentParts parts_within(SegmentParts p, int slots, int splits, int prefix_rows, int rows) {
  p.first = within(p.first, 0, slots - 1);
  p.own = within(p.own, 0, (slots - p.first) / 2 + 1);
  p.prefix = within(p.prefix, 0, splits);
  p.row = within(p.row, 0, prefix_rows - rows);
  return p;
}

}  // namespace cudalm_hip

#endif
