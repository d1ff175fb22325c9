// Attention of one or a few new tokens of every sequence over its pages.
//
// The rows of a (sequence, key-value head) pair, its new tokens times the
// query heads of the group, are the 16 columns of the matrix products, so a
// key or value is read once for all of them:
//
//   S^T = K Q^T    (16x16x32: A = 16 tokens x 32 channels, B = 32 channels x 16 rows)
//   O^T += V^T P^T (A = 16 channels x 32 tokens, B = 32 tokens x 16 rows)
//
// Both A operands come from the cache straight into registers: a lane reads
// 16 bytes of a token's key row, and 16 bytes of V's eight interleaved tokens
// of one channel. Which token a row of the first product stands for is free:
// row m of half f is token 8 (m / 4) + 4 f + m % 4 of the tile of 32, so that
// the lane that holds scores of row n, tokens 8 a .. 8 a + 7 after two products
// is the lane whose operand of the second product wants just those. Nothing
// goes through LDS before the end.
//
// A workgroup of WV waves takes RT tiles of 16 rows and WV / RT slices of the tokens,
// which it joins in LDS. A call's tiles of 32 tokens, those of all
// sequences and heads in a row, are cut into as many equal ranges as workgroups
// run at once: sequences of any mix of lengths keep all of them busy to the end.
// A range may end inside a sequence; such parts go to the workspace and a second
// kernel joins them. Where parts of a tile per slice are too few to fill the chip,
// every sequence gets as many workgroups as the longest needs, with no search for
// the ranges' places.
//
// Bytes bound it: 8 query heads on 2 of 256 read 64 KB of keys and values for 32
// tokens and multiply 0.3 MFLOP with them. 64 sequences of up to 8192 tokens (678 MB):
// 127-133 us and 6 for the join, 5.1 TB/s together, what a 1 GiB copy reaches; counters
// show 708 MB fetched. Five new tokens of 16 sequences of up to 5001, 32 heads on 8 of
// 128, with weights (215 MB): 52-65 us (card to card) and 16 for join and weights. One
// sequence of 777 tokens: 9 us and 4, chains of loads (table, keys, products, join).

#include <cstdint>

#include "paged_device.h"

namespace cudalm_hip {
namespace {

constexpr int kTile = 32;      // tokens per step of a wave
constexpr int kTileShift = 5;
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
  static __device__ __forceinline__ int total(const DecodeArgs& a, int lane, int to = 0,
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
  __device__ __forceinline__ void load(const DecodeArgs& a, int lane) {
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
  __device__ __forceinline__ int find(const DecodeArgs& a, int lane, int g, int* tiles, int* first) {
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

// WV waves: RT tiles of rows, WV / RT slices. RANGES: equal ranges of all tiles, else
// fixed splits.
template <typename T, int D, int RT, int WV, bool RANGES>
__global__ __launch_bounds__(64 * WV, 2) void paged_decode_kernel(const DecodeArgs a) {
  constexpr int KK = D / 32, DT = D / 16, SL = WV / RT;
  constexpr int kPitch = D + 4;
  // The queries of a tile of rows in the order of the operands (registers are for what
  // is on its way from memory), later the sums of two waves.
  union Shared {
    u32x4_t q[RT][KK][64];
    float o[2][16 * kPitch];
  };
  __shared__ Shared shared;
  __shared__ float mlbuf[WV][2][16];
  __shared__ uint32_t badbuf[WV];
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
    const PagedTiles tiles = a.tiles_of(length);
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
      if (!a.scores || !real || t0 + kTile > a.score_pitch) return;
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
          const bool one = has && paged_sees(t0 + 8 * quarter + e, pos, a.window, a.sinks);
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
    const bool whole = begin == 0 && end == all;
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
                sees |= paged_sees(t0 + e, pos, a.window, a.sinks) ? 1u << e : 0u;
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
    const int segment = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int b = segment / per_seq, all = uniform(a.count_of(b));
    const int per = tiles_per_split(all, a.splits, a.least);
    const int begin = split * per, end = begin + per < all ? begin + per : all;
    if (begin < end) part(b, segment % per_seq, begin, end, all, blockIdx.x);
  } else {
    const int total = Segments::total(a, lane), per = tiles_per_group(a, total);
    if (blockIdx.x >= static_cast<unsigned>((total + per - 1) / per)) return;
    int g = blockIdx.x * per;
    const int stop = g + per < total ? g + per : total;
    Segments segments = {};
    segments.load(a, lane);
#pragma unroll 1
    while (g < stop) {
      int all, start;
      const int b = segments.find(a, lane, g, &all, &start);
      const int hz = uniform((g - start) / all), begin = g - start - hz * all;
      const int end = stop - g < all - begin ? begin + stop - g : all;
      part(b, hz, begin, end, all, 2 * blockIdx.x + (begin == 0));
      g += end - begin;
    }
  }
}

// Where the parts of a segment are in the workspace: part 0 at slot0, part s > 0 at
// slot1 + s * step. One part: the output holds the result.
struct Parts {
  size_t slot0, slot1;
  int count, step;

  __device__ __forceinline__ Parts(const DecodeArgs& a, int b, int h, int zr, int lane) {
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
    }
  }
  __device__ __forceinline__ size_t at(int s) const {
    return s ? slot1 + static_cast<size_t>(s) * step : slot0;
  }
};

// The first `join_groups` workgroups: CH x SW waves per row of a segment that has more
// than one part, out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. A wave takes 64
// channels and every SW-th part; D / 64 / CH workgroups make a row.
// The others: weights[t] (+)= sum over rows of 2^(score - M) / l, for four tokens of a
// (sequence, head) per thread, with the rows' M and l joined from the parts. Five new
// tokens of 16 sequences of up to 5001, 32 heads on 8 of 128: 16 us, where a kernel
// for each of the two took 10 + 10. A row's parts are walked by one lane, which many
// parts of few rows wait for: one sequence of 32768 tokens, 8 heads on 2 of 256, takes 61
// us with weights, 29 without.
template <typename T, int D, int CH, int SW>
__global__ __launch_bounds__(64 * CH * SW) void paged_finish_kernel(const DecodeArgs a,
                                                                    unsigned join_groups,
                                                                    float* weights, int add,
                                                                    int token_groups) {
  union Shared {
    struct {
      float o[SW][64 * CH], l[SW];
    } join;
    float ml[2][kMaxRows];
  };
  __shared__ Shared shared;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  if (blockIdx.x < join_groups) {
    constexpr int kGroups = D / 64 / CH;
    const int chunk = blockIdx.x % kGroups * CH + wave % CH, sw = wave / CH;
    const int row = blockIdx.x / kGroups % a.rows, bh = blockIdx.x / kGroups / a.rows;
    const int b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads, zr = row / a.part_rows;
    const Parts parts(a, b, h, zr, lane);
    if (parts.count == 1) return;
    auto at = [&](int s) { return parts.at(s) * a.part_rows + row - zr * a.part_rows; };
    float M = kLowest;
    for (int s = lane; s < parts.count; s += 64) M = fmaxf(M, a.part_ml[2 * at(s)]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    float acc = 0, l = 0;
#pragma unroll 8
    for (int s = sw; s < parts.count; s += SW) {
      const float w = exp2_fast(a.part_ml[2 * at(s)] - M);
      l += w * a.part_ml[2 * at(s) + 1];
      acc += joined(w, a.part_o[at(s) * D + chunk * 64 + lane]);
    }
    if (SW > 1) {
      shared.join.o[sw][wave % CH * 64 + lane] = acc;
      if (lane == 0 && wave % CH == 0) shared.join.l[sw] = l;
      __syncthreads();
      if (sw > 0) return;
      acc = l = 0;
#pragma unroll
      for (int w = 0; w < SW; ++w)
        acc += shared.join.o[w][wave % CH * 64 + lane], l += shared.join.l[w];
    }
    const float inv = 1.0f / l;
    const int j = row / a.group, heads = a.group * a.kv.kv_heads;
    uint16_t* y = static_cast<uint16_t*>(a.out) +
                  ((static_cast<size_t>(b) * a.new_tokens + j) * heads + h * a.group + row - j * a.group) * D;
    y[chunk * 64 + lane] = static_cast<uint16_t>(T::pack(l == 0.0f ? 0.0f : acc * inv, 0.0f));
    return;
  }
  const int id = blockIdx.x - join_groups, bh = id / token_groups;
  const int b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;
  const int length = a.kv.uniform_length(b);
  const int t0 = 4 * (id % token_groups * blockDim.x + threadIdx.x);  // four tokens each
  if (t0 - 4 * static_cast<int>(threadIdx.x) >= length) return;
  for (int zr = wave; zr < a.zrows; zr += CH * SW) {
    const Parts parts(a, b, h, zr, lane);
    const int row = zr * a.part_rows + lane;
    if (lane < a.part_rows && row < a.rows) {
      float M = kLowest, l = 0;
      if (parts.count == 1) {
        const float* ml = a.final_ml + 2 * (static_cast<size_t>(bh) * a.rows + row);
        M = ml[0], l = ml[1];
      } else {
        for (int s = 0; s < parts.count; ++s) M = fmaxf(M, a.part_ml[2 * (parts.at(s) * a.part_rows + lane)]);
        for (int s = 0; s < parts.count; ++s) {
          const float* ml = a.part_ml + 2 * (parts.at(s) * a.part_rows + lane);
          l += exp2_fast(ml[0] - M) * ml[1];
        }
      }
      shared.ml[0][row] = M;
      shared.ml[1][row] = l == 0.0f ? 0.0f : 1.0f / l;
    }
  }
  __syncthreads();
  const PagedTiles tiles = a.tiles_of(length);
  const int P = 1 << a.kv.page_shift;
  typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
  for (int t = t0; t < length; t += 4 * token_groups * blockDim.x) {
    const int page = a.kv.page(b, t >> a.kv.page_shift);
    if (page < 0) continue;
    const int tile = t >> kTileShift;
    f32x4_t w = {0, 0, 0, 0};
    if ((tile < tiles.sink_tiles || tile >= tiles.sink_tiles + tiles.from) &&
        ((tile + 1) << kTileShift) <= a.score_pitch) {
      const float* sp = a.scores + static_cast<size_t>(bh) * a.rows * a.score_pitch + t;
#pragma unroll 8
      for (int r = 0; r < a.rows; ++r) {
        const f32x4_t s = *reinterpret_cast<const f32x4_t*>(sp + static_cast<size_t>(r) * a.score_pitch);
        const float M = shared.ml[0][r], inv = shared.ml[1][r];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] += exp2_fast(s[e] - M) * inv;
      }
    }
    float* dst = weights + (static_cast<size_t>(page) * a.kv.kv_heads + h) * P + (t & (P - 1));
    if (t + 4 <= length) {
      f32x4_any_t* d = reinterpret_cast<f32x4_any_t*>(dst);
      *d = add ? *d + w : w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t + e < length) dst[e] = add ? dst[e] + w[e] : w[e];
    }
  }
}

// How a call is cut.
struct DecodePlan {
  int rows, rt, zrows, part_rows, groups, splits, least, score_pitch;
  bool single;  // eight waves for a segment, and no join
  long long segments;
  size_t o_bytes, ml_bytes, final_bytes, score_bytes;
  bool joins() const { return splits != 1; }
  size_t bytes() const { return o_bytes + ml_bytes + final_bytes + score_bytes; }
};

DecodePlan plan_of(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int new_tokens, int mode) {
  DecodePlan p;
  p.rows = new_tokens * (q->heads / kv->kv_heads);
  const int row_tiles = (p.rows + 15) / 16;
  p.rt = row_tiles > 2 ? 4 : row_tiles;
  p.zrows = (row_tiles + p.rt - 1) / p.rt;
  p.part_rows = 16 * p.rt < p.rows ? 16 * p.rt : p.rows;
  const int len = expected_len(kv, q->max_len), window = window_of(q);
  long long tiles = (len + kTile - 1) / kTile;
  if (window > 0) {
    const long long near = (static_cast<long long>(window) + new_tokens + kTile - 2) / kTile + 1 +
                           (sinks_of(q) + kTile - 1) / kTile;
    tiles = near < tiles ? near : tiles;
  }
  const size_t bh = static_cast<size_t>(kv->batch) * kv->kv_heads;
  p.segments = static_cast<long long>(bh) * p.zrows;
  p.least = 4 / p.rt;  // a tile for each slice
  const long long parts = (tiles + p.least - 1) / p.least;
  const int at_once = (kv->head_dim == 64 ? 4 : 2) * cu_count();
  size_t slots;
  // One CU reads some 40 GB/s; up to 330 KB that takes less than a second launch (8
  // sequences of 500 tokens, 32 query heads on 8 of 128: 12.6 us against 18.3; one of
  // 777 on 2 of 256, past it: 24.5 against 15).
  p.single = p.rt < 4 && tiles * p.rt * kv->head_dim <= 2560 && p.segments * parts <= at_once;
  if (p.single) {
    p.splits = 1;
    p.groups = 0;
    slots = 0;
  } else if (parts <= 1 || p.segments * parts <= at_once) {
    p.splits = parts > 1 ? static_cast<int>(parts) : 1;
    p.groups = 0;
    slots = p.splits > 1 ? static_cast<size_t>(p.segments) * p.splits : 0;
  } else {
    p.splits = 0;
    p.groups = at_once;
    slots = 2 * static_cast<size_t>(at_once);
  }
  slots *= p.part_rows;
  p.o_bytes = slots * kv->head_dim * 4;
  p.ml_bytes = (slots * 8 + 15) / 16 * 16;
  p.score_pitch = mode ? (len + kTile - 1) / kTile * kTile : 0;
  p.final_bytes = mode ? (bh * p.rows * 8 + 15) / 16 * 16 : 0;
  p.score_bytes = mode ? bh * p.rows * p.score_pitch * 4 : 0;
  return p;
}

template <typename T, int D>
int launch(const DecodeArgs& a, const DecodePlan& p, float* weights, int mode, hipStream_t stream) {
  const unsigned grid = p.groups ? p.groups : static_cast<unsigned>(p.segments * p.splits);
  auto kernel = p.groups ? paged_decode_kernel<T, D, 1, 4, true> : paged_decode_kernel<T, D, 1, 4, false>;
  if (p.rt == 2) kernel = p.groups ? paged_decode_kernel<T, D, 2, 4, true> : paged_decode_kernel<T, D, 2, 4, false>;
  if (p.rt == 4) kernel = p.groups ? paged_decode_kernel<T, D, 4, 4, true> : paged_decode_kernel<T, D, 4, 4, false>;
  int threads = 256;
  if (p.single && p.rt < 4) {
    kernel = p.rt == 1 ? paged_decode_kernel<T, D, 1, 8, false> : paged_decode_kernel<T, D, 2, 8, false>;
    threads = 512;
  }
  kernel<<<grid, threads, 0, stream>>>(a);
  if (!p.joins() && !mode) return launch_status();
  if (const int rc = launch_status()) return rc;
  // Few rows: all waves that help, a workgroup for 64 channels (one sequence of 32768
  // tokens: 8 us, 16 with the other form); else one per row.
  const unsigned rows = static_cast<unsigned>(a.kv.batch * a.kv.kv_heads * a.rows);
  const bool few = rows <= static_cast<unsigned>(cu_count());
  const unsigned join = !p.joins() ? 0 : few ? rows * (D / 64) : rows;
  threads = few ? 1024 : D;
  const int token_groups = (p.score_pitch + 4 * threads - 1) / (4 * threads);
  const unsigned all = join + (mode ? a.kv.batch * a.kv.kv_heads * token_groups : 0);
  const int add = mode == CUDALM_PAGED_WEIGHTS_ADD;
  if (few)
    paged_finish_kernel<T, D, 1, 16><<<all, 1024, 0, stream>>>(a, join, weights, add, token_groups);
  else
    paged_finish_kernel<T, D, D / 64, 1><<<all, D, 0, stream>>>(a, join, weights, add, token_groups);
  return launch_status();
}

template <typename T>
int launch_d(int D, const DecodeArgs& a, const DecodePlan& p, float* weights, int mode,
             hipStream_t stream) {
  return D == 64    ? launch<T, 64>(a, p, weights, mode, stream)
         : D == 128 ? launch<T, 128>(a, p, weights, mode, stream)
                    : launch<T, 256>(a, p, weights, mode, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int new_tokens, int mode) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (new_tokens < 1 || mode < 0 || mode > CUDALM_PAGED_WEIGHTS_ADD) return CUDALM_W4A16_EINVAL;
  if (static_cast<long long>(new_tokens) * (q->heads / kv->kv_heads) > kMaxRows)
    return CUDALM_W4A16_EINVAL;
  const DecodePlan p = plan_of(kv, q, new_tokens, mode);
  const long long bh = static_cast<long long>(kv->batch) * kv->kv_heads;
  // all tiles are numbered in 31 bits, and where the last workgroup's range would end
  const long long cap = (static_cast<long long>(kv->max_pages) * kv->page_size + kTile - 1) / kTile;
  const long long tiles = p.segments * (cap + 1);
  if (tiles + (p.groups ? tiles / p.groups + p.groups : 0) >= (1LL << 31)) return CUDALM_W4A16_ERANGE;
  // workgroups of up to 1024 threads; with weights, one per 256 or more tokens
  const long long work = bh * p.rows + (mode ? bh * (p.score_pitch / 256 + 1) : 0);
  if (p.segments >= kMaxGemmTiles || work >= kMaxGemmTiles / 4) return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

}  // namespace

int paged_decode_regs(int type, int D) {
  if (type == CUDALM_PAGED_BF16)
    return D == 64    ? regs_of(paged_decode_kernel<PagedBf16, 64, 1, 4, true>)
           : D == 128 ? regs_of(paged_decode_kernel<PagedBf16, 128, 1, 4, true>)
           : D == 256 ? regs_of(paged_decode_kernel<PagedBf16, 256, 1, 4, true>)
                      : -1;
  return D == 64    ? regs_of(paged_decode_kernel<PagedF16, 64, 1, 4, true>)
         : D == 128 ? regs_of(paged_decode_kernel<PagedF16, 128, 1, 4, true>)
         : D == 256 ? regs_of(paged_decode_kernel<PagedF16, 256, 1, 4, true>)
                    : -1;
}

}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_paged_decode_workspace_bytes(const cudalm_paged_kv* kv,
                                                      const cudalm_paged_query* q, int new_tokens,
                                                      int weights_mode) {
  if (check(kv, q, new_tokens, weights_mode) != CUDALM_W4A16_OK) return 0;
  return plan_of(kv, q, new_tokens, weights_mode).bytes();
}

extern "C" int cudalm_paged_decode(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                                   int new_tokens, int weights_mode, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check(kv, q, new_tokens, weights_mode)) return rc;
  if (!q->q || !q->out || (weights_mode && !kv->weights)) return CUDALM_W4A16_ENULL;
  const DecodePlan p = plan_of(kv, q, new_tokens, weights_mode);
  if (p.bytes()) {
    if (!workspace) return CUDALM_W4A16_ENULL;
    if (!aligned(workspace, 16)) return CUDALM_W4A16_EALIGN;
    if (workspace_bytes < p.bytes()) return CUDALM_W4A16_ERANGE;
  }
  DecodeArgs a = {};
  a.kv = view_of(kv);
  a.k = static_cast<const uint16_t*>(kv->k);
  a.v = static_cast<const uint16_t*>(kv->v);
  a.q = static_cast<const uint16_t*>(q->q);
  a.out = q->out;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (p.joins()) {
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + p.o_bytes);
  }
  if (weights_mode) {
    a.final_ml = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes);
    a.scores = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes + p.final_bytes);
  }
  a.token_stride = q->token_stride;
  a.head_stride = q->head_stride;
  a.scale_log2 = q->scale * kLog2e;
  a.new_tokens = new_tokens;
  a.group = q->heads / kv->kv_heads;
  a.rows = p.rows;
  a.zrows = p.zrows;
  a.part_rows = p.part_rows;
  a.groups = p.groups;
  a.splits = p.splits;
  a.least = p.least;
  a.window = window_of(q);
  a.sinks = sinks_of(q);
  a.score_pitch = p.score_pitch;
  return kv->type == CUDALM_PAGED_BF16
             ? launch_d<PagedBf16>(kv->head_dim, a, p, kv->weights, weights_mode, stream)
             : launch_d<PagedF16>(kv->head_dim, a, p, kv->weights, weights_mode, stream);
}
