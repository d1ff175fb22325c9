// Groups of sequences that begin with the same tokens, on the device (gfx950).
#ifndef CUDALM_PAGED_SHARED_H
#define CUDALM_PAGED_SHARED_H

#include "paged_device.h"

namespace cudalm_hip {

// Group g is sequences cu[g] .. cu[g + 1] - 1; its first tokens, shared[g] of them, are
// those in the pages of sequence cu[g].
struct SharedGroups {
  const int32_t* cu;
  const int32_t* shared;
  int count;

  // Where group g's sequences begin and end; false where they are none or not there.
  __device__ __forceinline__ bool sequences(int g, int batch, int* begin, int* end) const {
    *begin = load_uniform(cu + g);
    *end = load_uniform(cu + g + 1);
    return *begin >= 0 && *end > *begin && *end <= batch;
  }
  __device__ __forceinline__ int tokens(const PagedView& kv, int g) const {
    const int n = load_uniform(shared + g), cap = kv.max_pages << kv.page_shift;
    return n < 0 ? 0 : n < cap ? n : cap;
  }
  // Tokens of sequence b (a lane's, or all lanes') that are its group's, 0 where it is in
  // no group. Every lane looks at all groups: their bounds are wave-uniform loads that
  // do not wait for each other, where a search would be a chain of them.
  __device__ __forceinline__ int shared_of(const PagedView& kv, int b) const {
    int n = 0;
    for (int g = 0; g < count; ++g) {
      int begin, end;
      const bool real = sequences(g, kv.batch, &begin, &end);
      const int t = tokens(kv, g);
      if (real && b >= begin && b < end) n = t;
    }
    return n;
  }
};

// PagedTiles of the tokens lo .. hi - 1 alone: those of the sinks, then those from the
// earliest window's first token on.
struct PagedRange {
  int base, sink_tiles, from, count;

  __device__ __forceinline__ PagedRange(int lo, int hi, int first, int last, int window, int sinks,
                                        int tile_shift) {
    const int mask = (1 << tile_shift) - 1;
    const int top = last + 1 < hi ? last + 1 : hi;
    base = lo >> tile_shift;
    int end = (top + mask) >> tile_shift;
    if (top <= lo || end < base) end = base;
    sink_tiles = 0;
    from = base;
    if (window > 0 && first - window + 1 > 0) {
      int st = ((sinks < hi ? sinks : hi) + mask) >> tile_shift, w = (first - window + 1) >> tile_shift;
      st = st < base ? base : st < end ? st : end;
      w = w < end ? w : end;
      if (w > st) sink_tiles = st - base, from = w - sink_tiles;
    }
    count = end - from;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i + base : i + from; }
};

}  // namespace cudalm_hip

#endif
