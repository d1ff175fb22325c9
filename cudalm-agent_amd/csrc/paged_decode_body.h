// Attention of a few new tokens of every sequence over ranges of its cached ones, and
// where the parts of a result are: what decode and decode with shared prefixes have in
// common (gfx950). How it works stands before the kernels.
#ifndef CUDALM_PAGED_DECODE_BODY_H
#define CUDALM_PAGED_DECODE_BODY_H

#include <type_traits>

#include "paged_shared.h"

namespace cudalm_hip {
namespace {

constexpr int kMaxRows = 1024;  // new tokens x query heads of a key-value head

// (sequence, head, 64 rows) in this order are the segments of a call.
struct DecodeArgs {
  PagedView kv;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  void* out;
  float* part_o;    // [parts][part_rows][D], part 2 w + x being workgroup w's ..
  float* part_ml;   // [parts][part_rows][2] .. or, with fixed splits, w itself
  float* final_ml;  // [bh][rows][2] or NULL
  float* scores;    // [bh][rows][score_pitch] (times scale log2 e) or NULL
  long long token_stride, head_stride;
  float scale_log2;
  int new_tokens, group, rows, zrows, part_rows, groups, splits, least, window, sinks, score_pitch;

  __device__ __forceinline__ PagedTiles tiles_of(int length) const {
    return PagedTiles(length, length - new_tokens, length - 1, window, sinks, kTileShift);
  }
  // Tiles of sequence b's segments; one where there are none, for its zeros.
  __device__ __forceinline__ int count_of(int b) const {
    const int n = tiles_of(kv.length(b)).count;
    return n > 0 ? n : 1;
  }
};

// The same where a sequence's first tokens are its group's, which others count: its own
// ones only.
struct OwnDecodeArgs : DecodeArgs {
  SharedGroups sharing;

  __device__ __forceinline__ PagedRange tiles_of(int length, int from) const {
    return PagedRange(from, length, length - new_tokens, length - 1, window, sinks, kTileShift);
  }
  __device__ __forceinline__ int count_of(int b) const {
    const int n = tiles_of(kv.length(b), sharing.shared_of(kv, b)).count;
    return n > 0 ? n : 1;
  }
};

// 16 bytes; `once`: nothing else of the call reads them, so the caches need not keep
// them (64 sequences of up to 3000 tokens, 8 heads of 128: 103 us without, 93 with).
template <bool once>
__device__ __forceinline__ u32x4_t load_once(const uint16_t* p) {
  const u32x4_t* q = reinterpret_cast<const u32x4_t*>(p);
  return once ? __builtin_nontemporal_load(q) : *q;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum of v over the wave's lanes.
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) v += __shfl_xor(v, x);
  return uniform(v);
}

// Where the segments lie in the row of all tiles (fewer than 2^31): 64 sequences at a
// time, a lane each.
struct Segments {
  int block, base;  // first sequence of the 64, tiles before it
  int count, end;   // this lane's sequence: tiles of a segment, end of its last one

  // Tiles of all sequences, and of those before sequence `to`.
  template <typename Args>
  static __device__ __forceinline__ int total(const Args& a, int lane, int to = 0,
                                              int* before = nullptr) {
    int all = 0, some = 0;
    for (int b = lane; b < a.kv.batch; b += 64) {
      const int n = a.count_of(b);
      all += n;
      some += b < to ? n : 0;
    }
    if (before) *before = wave_sum(some) * a.kv.kv_heads * a.zrows;
    return wave_sum(all) * a.kv.kv_heads * a.zrows;
  }
  template <typename Args>
  __device__ __forceinline__ void load(const Args& a, int lane) {
    count = block + lane < a.kv.batch ? a.count_of(block + lane) : 0;
    end = count * a.kv.kv_heads * a.zrows;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int o = __shfl_up(end, x);
      if (lane >= x) end += o;
    }
  }
  // The sequence of tile g (not before the block, and before the last), its tiles per
  // segment and the place of its first one.
  template <typename Args>
  __device__ __forceinline__ int find(const Args& a, int lane, int g, int* tiles, int* first) {
    for (;;) {
      const uint64_t after = __ballot(base + end > g);
      if (after) {
        const int x = __builtin_ctzll(after);
        *tiles = __builtin_amdgcn_readlane(count, x);
        *first = base + __builtin_amdgcn_readlane(end, x) - *tiles * a.kv.kv_heads * a.zrows;
        return block + x;
      }
      base += __builtin_amdgcn_readlane(end, 63);
      block += 64;
      load(a, lane);
    }
  }
};

// Tiles per workgroup.
__device__ __forceinline__ int tiles_per_group(const DecodeArgs& a, int total) {
  const int r = uniform((total + a.groups - 1) / a.groups);
  return r > a.least ? r : a.least;
}

// LDS of a workgroup of WV waves, RT tiles of rows: the queries of a tile of rows in the
// order of the operands (registers are for what is on its way from memory), later the
// sums of two waves.
template <int D, int RT, int WV>
struct DecodeLds {
  union {
    u32x4_t q[RT][D / 32][64];
    float o[2][16 * (D + 4)];
  } shared;
  float mlbuf[WV][2][16];
  uint32_t badbuf[WV];
};

// WV waves: RT tiles of rows, WV / RT slices. RANGES: equal ranges of all tiles, else
// fixed splits. Workgroup `block` of its call.
template <typename T, int D, int RT, int WV, bool RANGES, typename Args>
__device__ __forceinline__ void paged_decode_body(const Args& a, DecodeLds<D, RT, WV>& lds,
                                                  unsigned block) {
  constexpr bool kOwn = std::is_same<Args, OwnDecodeArgs>::value;
  constexpr int KK = D / 32, DT = D / 16, SL = WV / RT;
  constexpr int kPitch = D + 4;
  auto& shared = lds.shared;
  auto& mlbuf = lds.mlbuf;
  auto& badbuf = lds.badbuf;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 15, quarter = lane >> 4;
  const int rt = wave % RT, slice = wave / RT;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = (static_cast<size_t>(P) * D) * a.kv.kv_heads;
  const int ktok = 8 * (n >> 2) + (n & 3);  // token of K row n in half 0

  // tiles [begin, end) of a segment with `all` of them; `slot` of the workspace
  auto part = [&](int b, int hz, int begin, int end, int all, int slot) {
    const int h = hz / a.zrows, zr = hz % a.zrows;
    const int length = a.kv.uniform_length(b), first = length - a.new_tokens;
    int from = 0;  // tokens before it are another's to count
    if constexpr (kOwn) from = uniform(a.sharing.shared_of(a.kv, b));
    const auto tiles = [&] {
      if constexpr (kOwn)
        return a.tiles_of(length, from);
      else
        return a.tiles_of(length);
    }();
    auto row_sees = [&](int t, int pos) {
      return (!kOwn || t >= from) && paged_sees(t, pos, a.window, a.sinks);
    };
    // this lane's row
    const int row = (zr * RT + rt) * 16 + n;
    const bool real = row < a.rows;
    const int j = row / a.group;
    const int pos = real ? first + j : -1;
    if (slice == 0) {
      const uint16_t* qp =
          a.q +
          (static_cast<long long>(b) * a.new_tokens + (real ? j : 0)) * a.token_stride +
          (static_cast<long long>(h) * a.group + (real ? row - j * a.group : 0)) * a.head_stride +
          8 * quarter;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        u32x4_t v = *reinterpret_cast<const u32x4_t*>(qp + 32 * kk);
        if (!real) v = u32x4_t{0, 0, 0, 0};
        shared.q[rt][kk][lane] = v;
      }
      if (SL == 1) wave_lds_sync();
    }
    if (SL > 1) __syncthreads();
    const size_t head_elems = static_cast<size_t>(P) * D * h;
    f32x4_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_t{0, 0, 0, 0};
    float m = kLowest, l = 0;
    uint32_t bad = 0;
    u32x4_t kf[2][KK], vf[DT];

    // The next 32 tiles of this wave: lanes 2 i and 2 i + 1 hold the halves of tile i.
    int tile = 0;            // first token
    uint64_t half_at = 0;    // of the half's first key, and value, in its cache
    auto place = [&](int x) { return readlane64(half_at, x); };
    auto load_k = [&](int x) {
      const uint64_t at0 = place(x), at1 = place(x + 1), at = n < 8 ? at0 : at1;
      const uint16_t* kp = a.k + at + static_cast<uint32_t>((ktok & 15) * D + 8 * quarter);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int f = 0; f < 2; ++f)
          kf[f][kk] = load_once<RT == 1>(kp + 4 * f * D + 32 * kk);
    };
    auto load_v = [&](int x) {
      const uint64_t at0 = place(x), at1 = place(x + 1), at = quarter < 2 ? at0 : at1;
      const uint16_t* vp = a.v + at + static_cast<uint32_t>(8 * (quarter & 1) * D + 8 * n);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vf[dt] = load_once<RT == 1>(vp + 128 * dt);
    };
    float t[8];  // this lane's scores: its row, tokens 8 quarter .. 8 quarter + 7
    auto scores = [&]() {
      f32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
      asm volatile("" ::: "memory");  // the queries stay in LDS between tiles
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const u32x4_t qf = shared.q[rt][kk][lane];
        s0 = T::mfma(kf[0][kk], qf, s0);
        s1 = T::mfma(kf[1][kk], qf, s1);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t[e] = s0[e] * a.scale_log2;
        t[4 + e] = s1[e] * a.scale_log2;
      }
    };
    auto keep_scores = [&](int t0) {
      if (kOwn || !a.scores || !real || t0 + kTile > a.score_pitch) return;
      float* sp = a.scores +
                  (static_cast<size_t>(b * a.kv.kv_heads + h) * a.rows + row) * a.score_pitch + t0 +
                  8 * quarter;
      *reinterpret_cast<f32x4_t*>(sp) = f32x4_t{t[0], t[1], t[2], t[3]};
      *reinterpret_cast<f32x4_t*>(sp + 4) = f32x4_t{t[4], t[5], t[6], t[7]};
    };
    u32x4_t pf;
    auto softmax = [&]() {
      float top = t[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, t[e]);
      top = max_across_32(max_across_16(top));
      // The maximum may lag by up to 2^8: weights stay below 256, which neither
      // fp32 sums nor 16-bit weights mind, and most tiles rescale nothing.
      if (__any(top > m + 8.0f)) {
        const float next = fmaxf(m, top), r = exp2_fast(m - next);
        l *= r;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= r;
        m = next;
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = exp2_fast(t[e] - m), p1 = exp2_fast(t[e + 1] - m);
        l += p0 + p1;
        // The weights are rounded to the values' type, as the matrix unit takes
        // them; their sum l is that of the unrounded ones.
        pf[e / 2] = T::pack(p0, p1);
      }
    };

#pragma unroll 1
    for (int c = begin + slice; c < end; c += 32 * SL) {
      const int mine = c + SL * (lane >> 1);
      tile = tiles.tile(mine) << kTileShift;
      const int half_t = tile + 16 * (lane & 1);
      int page = -1;
      if (mine < end) page = a.kv.page(b, half_t >> a.kv.page_shift);
      half_at = static_cast<uint64_t>(page < 0 ? 0 : page) * page_elems + head_elems +
                static_cast<uint64_t>(half_t & (P - 1)) * D;
      const uint64_t here = __ballot(page >= 0);
      const int last = (end - c + SL - 1) / SL < 32 ? (end - c + SL - 1) / SL : 32;
      // The next tile's keys load while this one's weights are made, its values
      // while the scores are. Every tile is masked, and Inf and NaN taken out of its
      // values: at 5 TB/s each of 2048 waves gets a tile of 256 channels (32 KB) every
      // 13 us, and that is some hundred instructions.
      load_k(0);
#pragma unroll 1
      for (int x = 0; x < last; ++x) {
        load_v(2 * x);
        const int t0 = __builtin_amdgcn_readlane(tile, 2 * x);
        scores();
        if (x + 1 < last) load_k(2 * x + 2);
        const bool has = (here >> (2 * x + (quarter >> 1))) & 1;
        uint32_t sees = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool one = has && row_sees(t0 + 8 * quarter + e, pos);
          sees |= one ? 1u << e : 0u;
          t[e] = one ? t[e] : -__builtin_inff();
        }
        keep_scores(t0);
        softmax();
        // Zero weights times Inf or NaN are NaN: values of tokens that no row here
        // sees, which may be anything, are cleared, and Inf and NaN taken out of the
        // others; the rows that do see those get them at the end.
        uint32_t some = sees;
#pragma unroll
        for (int y = 1; y < 16; y <<= 1) some |= __shfl_xor(static_cast<int>(some), y);
        uint32_t keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          keep[w] = ((some >> (2 * w)) & 1 ? 0xFFFFu : 0u) | ((some >> (2 * w + 1)) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
          for (int w = 0; w < 4; ++w) vf[dt][w] &= keep[w];
          bad |= special_bits<T>(vf[dt]);
          o[dt] = T::mfma(finite_part<T>(vf[dt]), pf, o[dt]);
        }
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // join the slices: the upper half of the waves hands its sums down
    if (SL > 1) {
      if (quarter == 0) mlbuf[wave][0][n] = m, mlbuf[wave][1][n] = l;
      badbuf[wave] = __any(bad != 0);
      __syncthreads();
      float top = m;
#pragma unroll
      for (int s = 0; s < SL; ++s) top = fmaxf(top, mlbuf[s * RT + rt][0][n]);
      l = 0;
#pragma unroll
      for (int s = 0; s < SL; ++s)
        l += mlbuf[s * RT + rt][1][n] * exp2_fast(mlbuf[s * RT + rt][0][n] - top);
      const float r = exp2_fast(m - top);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= r;
      m = top;
      // the last one or two slices that still have sums add them to those before
      constexpr int kHands = 2 / RT > 0 ? 2 / RT : 1;
#pragma unroll
      for (int left = SL; left > 1;) {
        const int hands = kHands < left / 2 ? kHands : left / 2;
        if (slice >= left - hands && slice < left) {
          float* p = shared.o[(slice - left + hands) * RT + rt] + n * kPitch + 4 * quarter;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(p + 16 * dt) = o[dt];
        }
        __syncthreads();
        if (slice >= left - 2 * hands && slice < left - hands) {
          const float* p = shared.o[(slice - left + 2 * hands) * RT + rt] + n * kPitch + 4 * quarter;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] += *reinterpret_cast<const f32x4_t*>(p + 16 * dt);
        }
        __syncthreads();
        left -= hands;
      }
    }
    // to the workspace, or the output if the segment is all here
    const bool whole = !kOwn && begin == 0 && end == all;
    const int heads = a.group * a.kv.kv_heads;
    float* part_o = nullptr;
    uint16_t* out = nullptr;
    if (whole) {
      const size_t to = (static_cast<size_t>(b) * a.new_tokens + j) * heads + h * a.group + row - j * a.group;
      out = static_cast<uint16_t*>(a.out) + to * D + 4 * quarter;
    } else {
      part_o = a.part_o + (static_cast<size_t>(slot) * a.part_rows + rt * 16 + n) * D + 4 * quarter;
    }
    if (slice == 0 && real) {
      if (!whole) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(part_o + 16 * dt) = o[dt];
        if (quarter == 0) {
          float* ml = a.part_ml + 2 * (static_cast<size_t>(slot) * a.part_rows + rt * 16 + n);
          ml[0] = m, ml[1] = l;
        }
      } else {
        if (a.final_ml && quarter == 0) {
          float* ml = a.final_ml + 2 * (static_cast<size_t>(b * a.kv.kv_heads + h) * a.rows + row);
          ml[0] = m, ml[1] = l;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<u32x2_t*>(out + 16 * dt) = u32x2_t{
              T::pack(o[dt][0] * inv, o[dt][1] * inv), T::pack(o[dt][2] * inv, o[dt][3] * inv)};
      }
    }
    // Inf and NaN that were taken out, for the rows that see them: one wave after the
    // other adds Inf or -Inf to the sums.
    uint32_t any_bad = __any(bad != 0);
    if (SL > 1)
      for (int w = 0; w < WV; ++w) any_bad |= badbuf[w];
    if (any_bad) {
#pragma unroll 1
      for (int turn = 0; turn < SL; ++turn) {
        if (SL > 1) __syncthreads();
        if (turn != slice || !__any(bad != 0)) continue;
#pragma unroll 1
        for (int dt = 0; dt < DT; ++dt) {
          // how many tokens that a row sees hold +Inf or NaN, -Inf or NaN
          f32x4_t up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll 1
          for (int i = begin + slice; i < end; i += SL) {
            const int t0 = (tiles.tile(i) << kTileShift) + 8 * quarter;
            const int page = a.kv.page(b, t0 >> a.kv.page_shift);
            uint32_t sees = 0;
            u32x4_t v = {0, 0, 0, 0};
            if (page >= 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                sees |= row_sees(t0 + e, pos) ? 1u << e : 0u;
              v = *reinterpret_cast<const u32x4_t*>(a.v + page * page_elems + head_elems +
                                                    static_cast<size_t>(t0 & (P - 1)) * D + 8 * n +
                                                    128 * dt);
            }
            const u32x4_t ones = seen_operand<T>(sees);
            up = T::mfma(special_part<T>(v, ~0u), ones, up);
            down = T::mfma(special_part<T>(v, 0), ones, down);
          }
          if (!real || (whole && l == 0.0f)) continue;  // (no weight at all: zeros)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float add = (up[e] > 0 ? __builtin_inff() : 0.0f) + (down[e] > 0 ? -__builtin_inff() : 0.0f);
            if (whole)
              out[16 * dt + e] = static_cast<uint16_t>(T::pack(T::value(out[16 * dt + e]) + add, 0.0f));
            else
              part_o[16 * dt + e] += add;
          }
        }
      }
      if (SL > 1) __syncthreads();
    }
  };

  const int per_seq = a.kv.kv_heads * a.zrows;
  if constexpr (!RANGES) {
    const int segment = block / a.splits, split = block % a.splits;
    const int b = segment / per_seq, all = uniform(a.count_of(b));
    const int per = tiles_per_split(all, a.splits, a.least);
    const int begin = split * per, end = begin + per < all ? begin + per : all;
    if (begin < end) part(b, segment % per_seq, begin, end, all, block);
  } else {
    const int total = Segments::total(a, lane), per = tiles_per_group(a, total);
    if (block >= static_cast<unsigned>((total + per - 1) / per)) return;
    int g = block * per;
    const int stop = g + per < total ? g + per : total;
    Segments segments = {};
    segments.load(a, lane);
#pragma unroll 1
    while (g < stop) {
      int all, start;
      const int b = segments.find(a, lane, g, &all, &start);
      const int hz = uniform((g - start) / all), begin = g - start - hz * all;
      const int end = stop - g < all - begin ? begin + stop - g : all;
      // (a segment that is all here has a place of its own where that is not the output)
      const int slot = kOwn && end - begin == all ? 2 * a.groups + b * per_seq + hz : 2 * block + (begin == 0);
      part(b, hz, begin, end, all, slot);
      g += end - begin;
    }
  }
}

// Where the parts of a segment are in the workspace: part 0 at slot0, part s > 0 at
// slot1 + s * step. One part: the output holds the result.
struct Parts {
  size_t slot0, slot1;
  int count, step;

  template <typename Args>
  __device__ __forceinline__ Parts(const Args& a, int b, int h, int zr, int lane) {
    const int all = uniform(a.count_of(b));
    if (a.splits) {
      const int per = tiles_per_split(all, a.splits, a.least);
      count = (all + per - 1) / per;
      slot0 = slot1 = (static_cast<size_t>(b * a.kv.kv_heads + h) * a.zrows + zr) * a.splits;
      step = 1;
    } else {
      // workgroups w0 .. w1; their first parts, but for the first one's last
      int before;
      const int per = tiles_per_group(a, Segments::total(a, lane, b, &before));
      const int start = before + (h * a.zrows + zr) * all;
      const int w0 = start / per, w1 = (start + all - 1) / per;
      count = w1 - w0 + 1;
      slot0 = 2 * static_cast<size_t>(w0) + 1;
      slot1 = slot0 - 1;
      step = 2;
      if (std::is_same<Args, OwnDecodeArgs>::value && count == 1)
        slot0 = 2 * static_cast<size_t>(a.groups) + (static_cast<size_t>(b) * a.kv.kv_heads + h) * a.zrows + zr;
    }
  }
  __device__ __forceinline__ size_t at(int s) const {
    return s ? slot1 + static_cast<size_t>(s) * step : slot0;
  }
};

}  // namespace
}  // namespace cudalm_hip

#endif
