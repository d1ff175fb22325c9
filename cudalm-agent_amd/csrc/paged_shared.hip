// Attention of one or a few new tokens of every sequence, where groups of sequences
// begin with the same tokens.
//
// A group's queries, those of all its sequences, are the rows of one product over its
// shared tokens, so a shared key or value is fetched once for 128 of them; every
// sequence's own tokens are multiplied with its own queries. Both kinds of work leave
// sums under a running maximum in parts, which a last kernel joins:
//
//   out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s     over the parts of both kinds
//
// They share one launch: prefixes are bound by the matrix unit and their waits, own tokens by
// memory, so they run side by side on a CU (64 sequences behind 8192 tokens, 700 of their own each,
// 8 heads on 2 of 256: 20 us of prefixes and 20 of own tokens take 24.4 together, 102 MB; in
// launches of their own 22.6 and 24.3). The products are those of prefill and decode: which
// token a row of the first one stands for is free, so that a lane's scores are its operand of
// the second one.

#include <cmath>
#include <type_traits>

#include "paged_device.h"
#include "paged_places.h"

namespace cudalm_hip {
namespace {

constexpr int kTile = 32;  // tokens per step
constexpr int kTileShift = 5;
constexpr int kWaves = 4;  // of a workgroup
constexpr int kRows = 32 * kWaves;
constexpr int kMaxRows = 1024;  // new tokens x query heads of a key-value head

// Workgroups of a CU, and the tiles of keys or values that one has room for.
template <int D>
constexpr int kPerCu = D == 256 ? 2 : D == 128 ? 3 : 4;
template <int D>
constexpr int kRing = D == 256 ? 5 : D == 128 ? 6 : 8;
template <int D>
constexpr size_t kLdsBytes = static_cast<size_t>(kRing<D>) * kTile * D * 2;

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

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
    return clamped(kv, load_uniform(shared + g));
  }
  __device__ __forceinline__ static int clamped(const PagedView& kv, int n) {
    const int cap = kv.max_pages << kv.page_shift;
    return n < 0 ? 0 : n < cap ? n : cap;
  }
};

// The tiles of the tokens lo .. hi - 1 that some query of positions first .. last sees:
// those of the sinks, then those from the earliest window's first token on.
struct PagedRange {
  int base, sink_tiles, from, count;

  __device__ __forceinline__ PagedRange(int lo, int hi, int first, int last, int window, int sinks) {
    const int mask = kTile - 1, top = last + 1 < hi ? last + 1 : hi;
    base = lo >> kTileShift;
    const int end = top > lo ? (top + mask) >> kTileShift : base;
    sink_tiles = 0;
    from = base;
    if (window > 0 && first - window + 1 > 0) {
      int st = ((sinks < hi ? sinks : hi) + mask) >> kTileShift, w = (first - window + 1) >> kTileShift;
      st = st < base ? base : st < end ? st : end;
      w = w < end ? w : end;
      if (w > st) sink_tiles = st - base, from = w - sink_tiles;
    }
    count = end - from;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i + base : i + from; }
};

// Into how many parts a prefix of `tiles` tiles is cut: at most `splits`, of `least` tiles
// or more.
__device__ __forceinline__ int prefix_parts(int tiles, int splits, int least) {
  const int per = tiles_per_split(tiles, splits, least);
  return (tiles + per - 1) / per;
}

struct SharedArgs {
  PagedView kv;
  SharedGroups sharing;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  uint16_t* out;
  long long token_stride, head_stride;
  float scale_log2;
  int negate;  // scale is negative: queries are negated and it is taken positive
  int new_tokens, heads, group, rows, window, sinks;
  // Prefixes: rows of all groups by kRows, a group's beginning a new unit; parts by blocks
  // of 32 rows, [splits][units * kWaves][kv_heads], in the order of the registers.
  f32x4_t* prefix_o;   // .. [D / 8][64 lanes]
  float2* prefix_ml;   // .. [32]
  int units, splits, least;
  // Own tokens: (sequence, head, 16 RT rows) are segments, their tiles in a row are cut into
  // equal ranges. Part 2 w + x is range w's; whole segments follow, one each.
  float* own_o;        // [parts][part_rows][D]
  float2* own_ml;      // [parts][part_rows]
  int4* places;        // per segment: first part, how many, parts of its prefix, row in prefixes
  int zrows, part_rows, ranges, own_least;
};

// --- prefixes ---------------------------------------------------------------------

// N times 16 bytes per lane from base[x / 2] (wave-uniform) + offset[x % 2] to LDS: lane
// i's of load x land at dst + 4096 x + 16 i. The compiler's builtin for it makes every
// later LDS read wait for all such loads, those of later tiles among them; here
// loads_landed() does the waiting. (m0 holds the LDS address for the instruction.)
template <int N>
__device__ __forceinline__ void load_lds16(const uint64_t* base, const uint32_t* offset, uint32_t dst) {
  uint32_t saved;
  if constexpr (N == 1)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(dst), "v"(offset[0]), "s"(base[0])
        : "memory");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\t"
        "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(dst), "v"(offset[0]), "s"(base[0]), "s"(base[1])
        : "memory", "scc");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
        "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %4\n\t"
        "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %5\n\t"
        "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(dst), "v"(offset[0]), "v"(offset[1]), "s"(base[0]), "s"(base[1])
        : "memory", "scc");
}

// This wave's loads have landed but for the last N; a barrier after it speaks for all waves.
template <int N>
__device__ __forceinline__ void loads_landed() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// All waves have read what they read from LDS, and come here.
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int swap_bits_2_3(int r) {
  return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
}

// Key row r has chunk c at place c ^ chunk_exchange(r): 16 rows of 64 channels lie in
// eight lines of 64 banks, two to a line, wider ones in one line or more each.
template <int D>
__device__ __forceinline__ int chunk_exchange(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}

// kRows rows of a group (a wave has 32 of them as the columns of 32x32x16 products) against
// a part of its shared tokens:
//
//   S^T = K Q^T     (A = 32 tokens x 16 channels, B = 16 channels x 32 rows)
//   O^T += V^T P^T  (A = 32 channels x 16 tokens, B = 16 tokens x 32 rows)
//
// Tiles of keys and of values take turns in a ring of kRing places in LDS, which they
// reach from the pages without passing registers: unit 2 i is the keys of tile i, unit 2 i +
// 1 its values. A place is loaded again as soon as all waves have read it, so that kRing - 1 units
// are on their way or waiting at any time. A tile takes 1.7 us where 256 channels have two
// workgroups on a CU, of which the matrix unit works 30% for each: the rest is waiting for LDS and
// the other wave's turn (32768 tokens, 128 samples, 8 heads on 2 of 256: 69 us beside 1024 own
// tokens of every sample, 0.5 PFLOP/s of the prefix's products, 271 MB). Parts of more tiles would
// save bytes and leave CUs idle.
// Row r of a tile of 32 keys in LDS is token r with bits 2 and 3 exchanged: then the
// eight scores that a lane holds of a row after the first product are those of eight
// consecutive tokens, which is its operand of the second.
template <typename T, int D>
__device__ __forceinline__ void prefix_body(const SharedArgs& a, uint16_t* lds, unsigned block) {
  constexpr int KT = kTile, KK = D / 16, DT = D / 32;
  constexpr int C = D / 8;              // 16-byte chunks of a key row
  constexpr int kUnit = KT * D;         // elements of a unit
  constexpr int kLoads = D / 64;        // 1 KB loads of a unit per wave
  constexpr int R = kRing<D>;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 31, half = lane >> 5;

  // The row tiles of the same keys and values stand 8 workgroups apart, in one XCD, one
  // after the other.
  const int hs = static_cast<int>(block) / 8 / a.units * 8 + static_cast<int>(block) % 8;
  const int unit = static_cast<int>(block) / 8 % a.units;
  if (hs >= a.kv.kv_heads * a.splits) return;
  const int h = hs % a.kv.kv_heads, split = hs / a.kv.kv_heads;
  const int g = sequence_of(a.sharing.cu, a.sharing.count, unit, a.rows, kRows, 1);
  int b, b_end;
  if (g < 0 || !a.sharing.sequences(g, a.kv.batch, &b, &b_end)) return;
  const int row0 = (unit - (b * a.rows / kRows + g)) * kRows, rows = (b_end - b) * a.rows;
  if (row0 < 0 || row0 >= rows) return;  // (below 0 where cu does not ascend)
  const int length = a.sharing.tokens(a.kv, g);
  const int parts = prefix_parts((length + KT - 1) >> kTileShift, a.splits, a.least);
  if (split >= parts) return;

  // this lane's row (rows past the last are copies of it), and the positions of the wave's
  // and the workgroup's first and last
  const int wave_row = row0 + 32 * wave, row = wave_row + n;
  const bool real = row < rows;
  const int token = (real ? row : rows - 1) / a.group;
  const int seq = b + token / a.new_tokens;
  const int pos = a.kv.length(seq) - a.new_tokens + token % a.new_tokens;
  u32x4_t qf[KK];
  {
    const uint16_t* qp = a.q + (static_cast<long long>(b) * a.new_tokens + token) * a.token_stride +
                         (static_cast<long long>(h) * a.group + (real ? row : rows - 1) - token * a.group) * a.head_stride +
                         8 * half;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = load16(qp + 16 * kk);
      if (a.negate) qf[kk] ^= 0x80008000u;
    }
  }
  int wave_first = pos, wave_last = pos;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    wave_first = min(wave_first, __shfl_xor(wave_first, x));
    wave_last = max(wave_last, __shfl_xor(wave_last, x));
  }
  wave_first = uniform(wave_first);
  wave_last = uniform(wave_last);
  int wg_first = wave_first, wg_last = wave_last;
  {
    int* seen = reinterpret_cast<int*>(lds);
    if (lane == 0) seen[2 * wave] = wave_first, seen[2 * wave + 1] = wave_last;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) wg_first = min(wg_first, seen[2 * w]), wg_last = max(wg_last, seen[2 * w + 1]);
    wg_first = uniform(wg_first);
    wg_last = uniform(wg_last);
    __syncthreads();
  }
  const PagedRange tiles(0, length, wg_first, wg_last, a.window, a.sinks);
  const int per = tiles_per_split(tiles.count, parts, 1);
  const int begin = split * per, end = begin + per < tiles.count ? begin + per : tiles.count;

  f32x16_t o[DT];
  float m = kLowest, l = 0;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = static_cast<size_t>(P) * D * a.kv.kv_heads;
  const size_t head_elems = static_cast<size_t>(P) * D * h;
  // A wave loads 1 KB pieces wave, wave + 4, .. of a unit; of a half's 16 tokens, two (D =
  // 256: one with each offset), one, or half of one. Key row r of piece 4 x + wave is r0 + x
  // 2048 / D: its token is that of r0 plus a number that all lanes share, and the exchange of its
  // chunks is the same for every x but for chunk bit 3 where D = 256.
  const int r0 = wave * (512 / D) + lane / C;
  const int v_piece = wave * 64;  // in channels of the tile's groups of eight tokens
  // bytes from the half's first key, value
  const uint32_t k_lane = 2 * (swap_bits_2_3(r0) % 16 * D + 8 * ((lane % C) ^ chunk_exchange<D>(r0)));
  const uint32_t v_lane = 16 * (v_piece % D + lane) + (v_piece / D % 2) * 16 * D;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + wave * 1024;
  const uint32_t k_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) +
                         2 * (n * D + 8 * (half ^ chunk_exchange<D>(n)));

  // every row from position `from` to `to` sees all of the tile at t
  auto seen_whole = [&](int t, int from, int to) {
    return t + KT <= length && t + KT - 1 <= from && (a.window <= 0 || t > to - a.window || t + KT - 1 < a.sinks);
  };
  // Places, pages and visibility of 32 tiles: lanes 2 i and 2 i + 1 hold the halves of tile
  // i, masks a bit each; and those of the 32 before, since loads run ahead of products.
  uint64_t k_at = 0;  // of the half's first key; its first value is as far from the first of all
  const uint64_t to_v = reinterpret_cast<uint64_t>(a.v) - reinterpret_cast<uint64_t>(a.k);
  struct Masks {
    uint64_t absent, whole, wg_whole;
    bool plain;  // all here, and seen by all rows
  } masks = {0, 0, 0, false}, old_masks = masks;
  int ahead = begin;  // the first tile of the 32
  auto look_ahead = [&](int i) {
    old_masks = masks;
    ahead = i;
    const int first_token = tiles.tile(i + lane / 2) << kTileShift, t = first_token + 16 * (lane & 1);
    const bool in = i + lane / 2 < end;
    int page = -1;
    if (in) page = a.kv.page(b, t >> a.kv.page_shift);
    // absent pages are hidden below; any page will do
    k_at = reinterpret_cast<uint64_t>(a.k) +
           2 * (max(page, 0) * page_elems + head_elems + static_cast<uint64_t>(t & (P - 1)) * D);
    masks.absent = __ballot(page < 0);
    masks.whole = __ballot(seen_whole(first_token, wave_first, wave_last));
    masks.wg_whole = __ballot(seen_whole(first_token, wg_first, wg_last));
    masks.plain = !__any(in && (page < 0 || !seen_whole(first_token, wg_first, wg_last)));
  };
  const int units = 2 * (end - begin);
  int into = 0;  // the place of the next unit
  auto issue = [&](int u) {
    const int x = u & 63;
    if (x == 0 && u > 0) look_ahead(begin + u / 2);
    const uint64_t more = x & 1 ? to_v : 0;
    uint64_t base[2];
    // (of 64 channels a wave has half of one half)
    base[0] = readlane64(k_at, kLoads == 1 ? (x & ~1) + wave / 2 : x & ~1) + more;
    base[1] = kLoads == 1 ? 0 : readlane64(k_at, x | 1) + more;
    uint32_t offset[2] = {x & 1 ? v_lane : k_lane, 0};
    asm volatile("" : "+v"(offset[0]));  // (the other is made here, not held in a register)
    offset[1] = x & 1 ? offset[0] + 16 * D : (offset[0] ^ 128) + 8 * D;
    load_lds16<kLoads>(base, offset, lds0 + into * (2 * kUnit));
    into = into + 1 == R ? 0 : into + 1;
  };
  // Unit u is there for all waves, and all have read unit u - 1. (The last ones wait for
  // all that is on its way.)
  auto arrive = [&](int u) {
    if (u + R <= units + 1)
      loads_landed<(R - 2) * kLoads>();
    else
      loads_landed<0>();
    barrier();
  };
  // Zero weights times Inf or NaN are NaN. So in a tile that some row sees only
  // part of, values past the end or of absent pages (which may be anything) are
  // cleared, and Inf and NaN among the others taken out; the rows that do see
  // those get them at the end.
  uint32_t special = 0;
  auto clean = [&](u32x4_t* vt, int t0, uint32_t absent) {
#pragma unroll 2
    for (int u = threadIdx.x; u < KT / 8 * D; u += 64 * kWaves) {
      const int group = u / D, t = t0 + 8 * group;
      const bool gone = (absent >> (group >> 1)) & 1;
      u32x4_t w = vt[u];
      if (gone || t + 8 > length) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (gone || t + 2 * e >= length) w[e] &= 0xFFFF0000u;
          if (gone || t + 2 * e + 1 >= length) w[e] &= 0x0000FFFFu;
        }
        vt[u] = w;
      }
      const uint32_t bad = special_bits<T>(w);
      special |= bad;
      if (bad) vt[u] = finite_part<T>(w);
    }
  };

  constexpr int kAhead = D == 256 ? 3 : 4;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0;
  // (Its wait for the table is one for the queries too: the compiler, which does not see the
  // loads to LDS, would else have the products of every tile wait for all of those.)
  look_ahead(begin);
  for (int u = 0; u < R - 1 && u < units; ++u) issue(u);
  int from = 0;  // the place of the next unit to be read
  auto walk = [&](auto multiplies) {
#pragma unroll 1
  for (int u = 0; u < units; u += 2) {
    const int tile = begin + u / 2;
    arrive(u);
    if (u - 1 + R < units) issue(u - 1 + R);
    int t0 = 0;
    uint32_t absent = 0;
    bool whole = true, wg_whole = true;
    if (!(tile < ahead ? old_masks.plain : masks.plain)) {
      const Masks now = tile < ahead ? old_masks : masks;
      const int bit = u & 63;
      t0 = tiles.tile(tile) << kTileShift;
      absent = static_cast<uint32_t>(now.absent >> bit) & 3;
      whole = !absent && ((now.whole >> bit) & 1);
      wg_whole = !absent && ((now.wg_whole >> bit) & 1);
    }
    f32x16_t s;
    if constexpr (multiplies) {
      // chunk (2 kk + half) ^ chunk_exchange of row n: kk only flips bits 5 .. of the place
      const uint32_t key = k_lds + from * (2 * kUnit);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        s = T::mfma32(*reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(key ^ (32 * kk)), qf[kk], s);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int kk = 0; kk < KK - kAhead; ++kk) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
      __builtin_amdgcn_s_setprio(0);
    }
    from = from + 1 == R ? 0 : from + 1;
    arrive(u + 1);
    if (u + R < units) issue(u + R);
    uint16_t* vt = lds + from * kUnit;
    if (!wg_whole) {
      clean(reinterpret_cast<u32x4_t*>(vt), t0, absent);
      barrier();
    }
    if constexpr (multiplies) {
      // s[e] is the score of token t0 + 16 (e / 8) + 8 half + e % 8
      if (!whole) {
        // token t is seen from p if 0 <= p - t < window, or if t is a sink up to p
        const uint32_t reach = a.window > 0 ? a.window : 0x7FFFFFFF;
        const int back = pos - t0 - 8 * half, room = length - t0 - 8 * half;
        const int sunk = t0 < a.sinks ? min(a.sinks - t0 - 8 * half, back + 1) : -1;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = 16 * (e >> 3) + (e & 7);
          const bool sees = (static_cast<uint32_t>(back - i) < reach || i < sunk) && i < room &&
                            !((absent >> (e >> 3)) & 1);
          s[e] = sees ? s[e] : -__builtin_inff();
        }
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top = max_across_32(top) * a.scale_log2;
      // The maximum may lag by up to 2^8: weights stay below 256, which neither fp32 sums nor
      // 16-bit weights mind, and most tiles rescale nothing.
      if (__any(top > m + 8.0f)) {
        const float next = fmaxf(m, top), r = exp2_fast(m - next);
        l *= r;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= r;
        m = next;
      }
      float sum = 0;
      const u32x4_t* vp = reinterpret_cast<const u32x4_t*>(vt) + half * D + n;
      u32x4_t pf[2];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = exp2_fast(__builtin_fmaf(s[e], a.scale_log2, -m));
        const float p1 = exp2_fast(__builtin_fmaf(s[e + 1], a.scale_log2, -m));
        sum += p0 + p1;
        // rounded to the values' type, as the matrix unit takes them; l sums the unrounded ones.
        // (Two numbers for each would double the second product; against 64 bits the results' error is
        // 0.0023 of their size in bf16, 0.0017 with exact weights: their own rounding.)
        pf[e / 8][e % 8 / 2] = T::pack(p0, p1);
      }
      l += sum;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < 2 * DT; ++x)
        o[x % DT] = T::mfma32(vp[(x / DT) * 2 * D + 32 * (x % DT)], pf[x / DT], o[x % DT]);
      if (D >= 128) {
        constexpr int kFirst = 1 + D / 128;
        __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
        for (int x = 0; x < 2 * DT - kFirst; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kFirst, 0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    from = from + 1 == R ? 0 : from + 1;
  }
  };
  const bool idle = wave_row >= rows;  // nothing to multiply
  if (idle)
    walk(std::false_type());
  else
    walk(std::true_type());
  // Inf or NaN for the sums of channels 32 dt .. whose rows see such a value: how many
  // tokens hold +Inf or NaN, -Inf or NaN. In tiles that were not cleaned a weight that
  // underflows has made NaN of Inf, so what the sums hold there does not count.
  auto add_special = [&](f32x16_t& r, int dt) {
    f32x16_t up, down;
#pragma unroll
    for (int e = 0; e < 16; ++e) up[e] = down[e] = 0;
#pragma unroll 1
    for (int i = begin; i < end; ++i) {
      const int place = tiles.tile(i) << kTileShift;
#pragma unroll 1
      for (int y = 0; y < KT / 16; ++y) {
        const int t = place + 16 * y + 8 * half;
        const int page = a.kv.page(b, t >> a.kv.page_shift);
        uint32_t seen = 0;
        u32x4_t w = {0, 0, 0, 0};
        if (page >= 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            seen |= t + e < length && paged_sees(t + e, pos, a.window, a.sinks) ? 1u << e : 0u;
          w = load16(a.v + page * page_elems + head_elems + static_cast<size_t>(t & (P - 1)) * D + 8 * (32 * dt + n));
        }
        const u32x4_t ones = seen_operand<T>(seen);
        up = T::mfma32(special_part<T>(w, ~0u), ones, up);
        down = T::mfma32(special_part<T>(w, 0), ones, down);
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (up[e] > 0 || down[e] > 0)
        r[e] = (up[e] > 0 ? __builtin_inff() : 0.0f) + (down[e] > 0 ? -__builtin_inff() : 0.0f);
  };
  f32x16_t most = o[0];  // of the sums' sizes, NaN if one of them is
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) most[e] = __builtin_elementwise_maximum(fabsf(most[e]), fabsf(o[dt][e]));
#pragma unroll
  for (int x = 8; x > 0; x >>= 1)
#pragma unroll
    for (int e = 0; e < x; ++e) most[e] = __builtin_elementwise_maximum(most[e], most[e + x]);
  barrier();  // the ring has been read: its first words hold the waves' votes
  uint32_t* votes = reinterpret_cast<uint32_t*>(lds);
  votes[wave] = __any(special != 0 || !(most[0] < __builtin_inff()));
  __syncthreads();
  special = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) special |= votes[w];
  special = uniform(special);
  if (idle) return;
  l += __shfl_xor(l, 32);
  const size_t at = (static_cast<size_t>(split) * (a.units * kWaves) + unit * kWaves + wave) * a.kv.kv_heads + h;
  // -inf tells the join that there is nothing to read: no weight here, nor Inf or NaN
  if (half == 0) a.prefix_ml[at * 32 + n] = float2{l == 0.0f && !special ? -__builtin_inff() : m, l};
  if (begin >= end) return;
  f32x4_t* p = a.prefix_o + at * (D / 8 * 64) + lane;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    f32x16_t r = o[dt];
    if (special) add_special(r, dt);
#pragma unroll
    for (int y = 0; y < 4; ++y)
      p[(4 * dt + y) * 64] = f32x4_t{r[4 * y], r[4 * y + 1], r[4 * y + 2], r[4 * y + 3]};
  }
}

// --- own tokens ---------------------------------------------------------------------

// 16 bytes; `once`: nothing else of the call reads them, so the caches need not keep them. (For
// values. Keys are read half a line at a time, and the caches have to keep the other half: 64
// sequences of 2000 own tokens, 8 heads of 128, take 90 us so, 104 with streaming loads for both and
// 113 with them for neither.)
template <bool once>
__device__ __forceinline__ u32x4_t load_once(const uint16_t* p) {
  const u32x4_t* q = reinterpret_cast<const u32x4_t*>(p);
  return once ? __builtin_nontemporal_load(q) : *q;
}

// Sequences' own tokens in the row of all tiles (fewer than 2^31), 64 sequences at a time, a
// lane each.
struct Segments {
  int block, base;   // first sequence of the 64, tiles before it
  int length, from;  // this lane's sequence: tokens, and how many of them are its group's
  int row;           // its first row among those of prefixes
  int count, end;    // tiles of a segment, end of its last one

  // Sequence b's group, 64 bounds of groups at a time: each lane looks for its place among those
  // that the others hold. (64 groups of four sequences, prefixes of 1024 of 128 channels: 35 us the
  // call; a walk of all lanes over the groups took 86.)
  __device__ __forceinline__ int group_of(const SharedArgs& a, int lane, int b) {
    int g = -1;
    for (int g0 = 0; g0 <= a.sharing.count; g0 += 64) {
      const int first = g0 + lane <= a.sharing.count ? a.sharing.cu[g0 + lane] : 0x7FFFFFFF;
      int n = 0;  // four times how many of them are not behind b
#pragma unroll
      for (int x = 32; x; x >>= 1) n += __builtin_amdgcn_ds_bpermute(n + 4 * x - 4, first) <= b ? 4 * x : 0;
      n += __builtin_amdgcn_readlane(first, 63) <= b ? 4 : 0;
      g += n / 4;
      if (!__any(n == 256)) break;
    }
    return g;
  }
  __device__ __forceinline__ void load(const SharedArgs& a, int lane) {
    asm volatile("" : "+v"(lane));  // nothing here is worth a register elsewhere
    const int b = block + lane, per_seq = a.kv.kv_heads * a.zrows;
    length = b < a.kv.batch ? a.kv.length(b) : 0;
    from = row = 0;
    const int g = group_of(a, lane, b);
    if (g >= 0 && g < a.sharing.count) {
      const int first = a.sharing.cu[g];
      if (first >= 0 && b >= first && b < a.sharing.cu[g + 1] && a.sharing.cu[g + 1] <= a.kv.batch) {
        from = a.sharing.clamped(a.kv, a.sharing.shared[g]);
        row = (first * a.rows / kRows + g) * kRows + (b - first) * a.rows;
      }
    }
    const PagedRange tiles(from, length, length - a.new_tokens, length - 1, a.window, a.sinks);
    count = b < a.kv.batch ? max(tiles.count, 1) : 0;  // (a place for the row's zeros)
    end = count * per_seq;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int o = __shfl_up(end, x);
      if (lane >= x) end += o;
    }
  }
  // The tiles of all sequences. Past 64 of them the waves of a workgroup share the work: `totals` gets
  // the tiles of every 64, of several such blocks where there are more than kTotals. (256 sequences of
  // 100 tokens behind one prefix: 21 us, 24.5 where every wave went through all of them.)
  static constexpr int kTotals = 4096;
  __device__ __forceinline__ int total(const SharedArgs& a, int lane, int wave, int* totals) {
    const int blocks = (a.kv.batch + 63) / 64, each = (blocks + kTotals - 1) / kTotals;
    base = block = 0;
    if (blocks == 1) {
      load(a, lane);
      return __builtin_amdgcn_readlane(end, 63);
    }
    const int entries = (blocks + each - 1) / each;
    for (int e = wave; e < entries; e += kWaves) {
      int all = 0;
      for (int i = e * each; i < blocks && i < (e + 1) * each; ++i) {
        block = 64 * i;
        load(a, lane);
        all += __builtin_amdgcn_readlane(end, 63);
      }
      if (lane == 0) totals[e] = all;
    }
    barrier();
    int all = 0;
    for (int e = 0; e < entries; e += 64) all += __builtin_amdgcn_readlane(sums(lane, totals, e, entries), 63);
    return all;
  }
  // The running sums of totals e .. e + 63.
  __device__ __forceinline__ static int sums(int lane, const int* totals, int e, int entries) {
    int sum = e + lane < entries ? totals[e + lane] : 0;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int o = __shfl_up(sum, x);
      if (lane >= x) sum += o;
    }
    return sum;
  }
  // Goes to the block of tile g (below total()).
  __device__ __forceinline__ void seek(const SharedArgs& a, int lane, const int* totals, int g) {
    const int blocks = (a.kv.batch + 63) / 64, each = (blocks + kTotals - 1) / kTotals;
    if (blocks == 1) return;
    base = 0;
    for (int e = 0, entries = (blocks + each - 1) / each;; e += 64) {
      const int sum = sums(lane, totals, e, entries);
      const uint64_t after = __ballot(base + sum > g);
      if (after) {
        const int x = __builtin_ctzll(after);
        if (x) base += __builtin_amdgcn_readlane(sum, x - 1);
        block = 64 * (e + x) * each;
        break;
      }
      base += __builtin_amdgcn_readlane(sum, 63);
    }
    load(a, lane);
  }
  // The lane whose sequence has tile g, not before the block; -1: none, where lengths change under the
  // call (the join then reads an entry of `places` that was not written, within its bounds).
  __device__ __forceinline__ int find(const SharedArgs& a, int lane, int g) {
    for (;;) {
      const uint64_t after = __ballot(base + end > g);
      if (after) return __builtin_ctzll(after);
      if (block + 64 >= a.kv.batch) return -1;
      base += __builtin_amdgcn_readlane(end, 63);
      block += 64;
      load(a, lane);
    }
  }
};

// The rows of a (sequence, head), its new tokens times the group's query heads, are the 16
// columns of 16x16x32 products; keys and values come straight from the pages into
// registers. RT tiles of 16 rows have a wave each, which walk over the same tokens; beside them
// 4 / RT ranges. No wave waits for another, since a range's end may be a wave's second part or
// third (barriers for them: 42 us above where there were 28 without). Alone they stream 45 MB in 20 us,
// 128 x 1024 tokens 134 MB in 37: memory and the first loads' chain (lengths, groups, pages, keys).
template <typename T, int D, int RT>
__device__ __forceinline__ void own_body(const SharedArgs& a, uint16_t* lds, unsigned block) {
  constexpr int KK = D / 32, DT = D / 16, SL = kWaves / RT;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 15, quarter = lane >> 4;
  const int rt = wave % RT, range = block * SL + wave / RT;
  // The queries in the order of the operands (registers are for what is on its way from
  // memory).
  u32x4_t* q_lds = reinterpret_cast<u32x4_t*>(lds) + wave * (KK * 64) + lane;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = (static_cast<size_t>(P) * D) * a.kv.kv_heads;
  const int ktok = 8 * (n >> 2) + (n & 3);  // token of K row n in half 0

  Segments segments;
  int* totals = reinterpret_cast<int*>(reinterpret_cast<u32x4_t*>(lds) + kWaves * KK * 64);
  static_assert(kWaves * KK * 1024 + 4 * Segments::kTotals <= kLdsBytes<D>, "the queries and the totals have room");
  const int total = segments.total(a, lane, wave, totals);
  int per = uniform((total + a.ranges - 1) / a.ranges);
  per = per > a.own_least ? per : a.own_least;
  if (static_cast<long long>(range) * per >= total) return;
  int g = range * per;
  segments.seek(a, lane, totals, g);
  const int stop = g + per < total ? g + per : total, per_seq = a.kv.kv_heads * a.zrows;
#pragma unroll 1
  while (g < stop) {
    const int x0 = segments.find(a, lane, g), b = segments.block + x0;
    if (x0 < 0) return;
    const int all = __builtin_amdgcn_readlane(segments.count, x0);
    const int start = segments.base + __builtin_amdgcn_readlane(segments.end, x0) - all * per_seq;
    const int hz = uniform((g - start) / all), h = hz / a.zrows, zr = hz % a.zrows;
    const int begin = g - start - hz * all, end = stop - g < all - begin ? begin + stop - g : all;
    const int length = __builtin_amdgcn_readlane(segments.length, x0), from = __builtin_amdgcn_readlane(segments.from, x0);
    const PagedRange tiles(from, length, length - a.new_tokens, length - 1, a.window, a.sinks);
    const int segment = b * per_seq + hz;
    const int slot = end - begin == all ? 2 * a.ranges + segment : 2 * range + (begin == 0);
    if (begin == 0 && rt == 0 && lane == 0)
      a.places[segment] = int4{slot, (g + all - 1) / per - range + 1,
                               prefix_parts((from + kTile - 1) >> kTileShift, a.splits, a.least),
                               __builtin_amdgcn_readlane(segments.row, x0)};
    // this lane's row
    const int row = (zr * RT + rt) * 16 + n;
    const bool real = row < a.rows;
    const int j = real ? row / a.group : 0;
    const int pos = real ? length - a.new_tokens + j : -1;
    const size_t head_elems = static_cast<size_t>(P) * D * h;
    auto row_sees = [&](int t) { return t >= from && paged_sees(t, pos, a.window, a.sinks); };
    // Pages of the next 32 tiles: lanes 2 i and 2 i + 1 hold the halves of tile i.
    int tile = 0, page = -1;  // first token
    uint64_t half_at = 0;     // of the half's first key, and value, in its cache
    auto look_up = [&](int c) {
      const int mine = c + (lane >> 1);
      tile = tiles.tile(mine) << kTileShift;
      page = -1;
      if (mine < end) page = a.kv.page(b, (tile + 16 * (lane & 1)) >> a.kv.page_shift);
    };
    look_up(begin);
    {
      const uint16_t* qp = a.q + (static_cast<long long>(b) * a.new_tokens + j) * a.token_stride +
                           (static_cast<long long>(h) * a.group + (real ? row - j * a.group : 0)) * a.head_stride +
                           8 * quarter;
      u32x4_t qf[KK];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[kk] = load16(qp + 32 * kk);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (!real) qf[kk] = u32x4_t{0, 0, 0, 0};
        if (a.negate) qf[kk] ^= 0x80008000u;
        q_lds[kk * 64] = qf[kk];
      }
    }
    f32x4_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_t{0, 0, 0, 0};
    float m = kLowest, l = 0;
    uint32_t bad = 0;
    u32x4_t kf[2][KK], vf[DT];
    auto place = [&](int x) { return readlane64(half_at, x); };
    auto load_k = [&](int x) {
      const uint64_t at0 = place(x), at1 = place(x + 1), at = n < 8 ? at0 : at1;
      const uint16_t* kp = a.k + at + static_cast<uint32_t>((ktok & 15) * D + 8 * quarter);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int f = 0; f < 2; ++f) kf[f][kk] = load16(kp + 4 * f * D + 32 * kk);
    };
    auto load_v = [&](int x) {
      const uint64_t at0 = place(x), at1 = place(x + 1), at = quarter < 2 ? at0 : at1;
      const uint16_t* vp = a.v + at + static_cast<uint32_t>(8 * (quarter & 1) * D + 8 * n);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vf[dt] = load_once<RT == 1>(vp + 128 * dt);
    };
#pragma unroll 1
    for (int c = begin; c < end; c += 32) {
      if (c > begin) look_up(c);
      half_at = static_cast<uint64_t>(page < 0 ? 0 : page) * page_elems + head_elems +
                static_cast<uint64_t>((tile + 16 * (lane & 1)) & (P - 1)) * D;
      const uint64_t here = __ballot(page >= 0);
      const int last = end - c < 32 ? end - c : 32;
      // The next tile's keys load while this one's weights are made, its values while the
      // scores are.
      load_k(0);
      wave_lds_sync();
#pragma unroll 1
      for (int x = 0; x < last; ++x) {
        load_v(2 * x);
        const int t0 = __builtin_amdgcn_readlane(tile, 2 * x);
        float t[8];  // this lane's scores: its row, tokens 8 quarter .. 8 quarter + 7
        {
          f32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
          asm volatile("" ::: "memory");  // the queries stay in LDS between tiles
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            const u32x4_t qf = q_lds[kk * 64];
            s0 = T::mfma(kf[0][kk], qf, s0);
            s1 = T::mfma(kf[1][kk], qf, s1);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            t[e] = s0[e] * a.scale_log2;
            t[4 + e] = s1[e] * a.scale_log2;
          }
        }
        if (x + 1 < last) load_k(2 * x + 2);
        const bool has = (here >> (2 * x + (quarter >> 1))) & 1;
        uint32_t sees = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool one = has && row_sees(t0 + 8 * quarter + e);
          sees |= one ? 1u << e : 0u;
          t[e] = one ? t[e] : -__builtin_inff();
        }
        float top = t[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, t[e]);
        top = max_across_32(max_across_16(top));
        if (__any(top > m + 8.0f)) {  // (a lagging maximum, as above)
          const float next = fmaxf(m, top), r = exp2_fast(m - next);
          l *= r;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] *= r;
          m = next;
        }
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float p0 = exp2_fast(t[e] - m), p1 = exp2_fast(t[e + 1] - m);
          l += p0 + p1;
          pf[e / 2] = T::pack(p0, p1);  // (rounded as in prefixes)
        }
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
    // Inf and NaN that were taken out, for the rows that see them: how many tokens hold
    // +Inf or NaN, -Inf or NaN.
    if (__any(bad != 0)) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x4_t up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll 1
        for (int i = begin; i < end; ++i) {
          const int t0 = (tiles.tile(i) << kTileShift) + 8 * quarter;
          const int at = a.kv.page(b, t0 >> a.kv.page_shift);
          uint32_t sees = 0;
          u32x4_t v = {0, 0, 0, 0};
          if (at >= 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sees |= row_sees(t0 + e) ? 1u << e : 0u;
            v = load16(a.v + at * page_elems + head_elems + static_cast<size_t>(t0 & (P - 1)) * D + 8 * n + 128 * dt);
          }
          const u32x4_t ones = seen_operand<T>(sees);
          up = T::mfma(special_part<T>(v, ~0u), ones, up);
          down = T::mfma(special_part<T>(v, 0), ones, down);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[dt][e] += (up[e] > 0 ? __builtin_inff() : 0.0f) + (down[e] > 0 ? -__builtin_inff() : 0.0f);
      }
    }
    if (real) {
      const size_t at = static_cast<size_t>(slot) * a.part_rows + rt * 16 + n;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4_t*>(a.own_o + at * D + 16 * dt + 4 * quarter) = o[dt];
      if (quarter == 0) a.own_ml[at] = float2{m, l};
    }
    wave_lds_sync();  // the queries have been read
    g += end - begin;
  }
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(64 * kWaves, kPerCu<D>) void paged_shared_kernel(const SharedArgs a, unsigned prefix_blocks) {
  extern __shared__ uint16_t shared_lds[];
  if (blockIdx.x < prefix_blocks)
    prefix_body<T, D>(a, shared_lds, blockIdx.x);
  else
    own_body<T, D, RT>(a, shared_lds, blockIdx.x - prefix_blocks);
}

// --- the join -------------------------------------------------------------------------

// 32 rows of a key-value head, PC pieces of eight channels; the WV waves of a workgroup take
// every WV-th part. A lane has the row n of a prefix's register order and four channels of a
// piece, so that a part's piece is one load of 1 KB. The maximum runs along, which saves a pass
// over the parts' maxima.
template <typename T, int D, int PC, int WV>
__global__ __launch_bounds__(64 * WV) void paged_shared_join_kernel(const SharedArgs a, int chunks) {
  constexpr int kAtOnce = 4;
  __shared__ f32x4_t sums[WV][PC][64];
  __shared__ float2 tops[WV][32];
  const int lane = threadIdx.x & 63, wave = wave_id(), n = lane & 31, half = lane >> 5;
  const int chunk = blockIdx.x % chunks, h = blockIdx.x / chunks % a.kv.kv_heads;
  const int R = static_cast<int>(blockIdx.x / chunks / a.kv.kv_heads) * 32 + n;
  const bool real = R < a.kv.batch * a.rows;
  const int b = (real ? R : 0) / a.rows, r = (real ? R : 0) - b * a.rows, zr = r / a.part_rows;
  const int4 entry = a.places[(b * a.kv.kv_heads + h) * a.zrows + zr];
  const SegmentParts place = parts_within({entry.x, entry.y, entry.z, entry.w},
                                          2 * a.ranges + a.kv.batch * a.kv.kv_heads * a.zrows, a.splits,
                                          a.units * kRows, a.rows);
  const int before = place.prefix, count = real ? before + place.own : 0, prow = place.row + r;
  f32x4_t acc[PC];
#pragma unroll
  for (int x = 0; x < PC; ++x) acc[x] = f32x4_t{0, 0, 0, 0};
  float m = kLowest, l = 0;
  for (int s0 = wave; __any(s0 < count); s0 += WV * kAtOnce) {
    float2 ml[kAtOnce];
    f32x4_t o[kAtOnce][PC];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = s0 + WV * i;
      ml[i] = float2{-__builtin_inff(), 0};
      if (s < before) {
        const size_t at = (static_cast<size_t>(s) * (a.units * kWaves) + prow / 32) * a.kv.kv_heads + h;
        ml[i] = a.prefix_ml[at * 32 + prow % 32];
#pragma unroll
        for (int x = 0; x < PC; ++x)
          o[i][x] = a.prefix_o[(at * (D / 8) + chunk * PC + x) * 64 + half * 32 + prow % 32];
      } else if (s < count) {
        const int y = s - before;
        const size_t at = static_cast<size_t>(own_part(place.first, y)) * a.part_rows + r - zr * a.part_rows;
        ml[i] = a.own_ml[at];
#pragma unroll
        for (int x = 0; x < PC; ++x)
          o[i][x] = *reinterpret_cast<const f32x4_t*>(a.own_o + at * D + 8 * (chunk * PC + x) + 4 * half);
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
    const float again = exp2_fast(m - top);
    m = top;
    l *= again;
#pragma unroll
    for (int x = 0; x < PC; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[x][e] = joined(again, acc[x][e]);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (ml[i].x == -__builtin_inff()) continue;  // nothing there
      const float w = exp2_fast(ml[i].x - m);
      l += w * ml[i].y;
#pragma unroll
      for (int x = 0; x < PC; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][e] += joined(w, o[i][x][e]);
    }
  }
#pragma unroll
  for (int x = 0; x < PC; ++x) sums[wave][x][lane] = acc[x];
  if (half == 0) tops[wave][n] = float2{m, l};
  __syncthreads();
  if (wave >= PC) return;
  float M = kLowest;
#pragma unroll
  for (int w = 0; w < WV; ++w) M = fmaxf(M, tops[w][n].x);
  l = 0;
  f32x4_t y = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < WV; ++w) {
    const float weight = exp2_fast(tops[w][n].x - M);
    l += weight * tops[w][n].y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += joined(weight, sums[w][wave][lane][e]);
  }
  if (!real) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0.0f : y[e] * inv;  // (no weight at all: zeros)
  const int j = r / a.group;
  const size_t to = (static_cast<size_t>(b) * a.new_tokens + j) * a.heads + h * a.group + r - j * a.group;
  *reinterpret_cast<u32x2_t*>(a.out + to * D + 8 * (chunk * PC + wave) + 4 * half) =
      u32x2_t{T::pack(y[0], y[1]), T::pack(y[2], y[3])};
}

// --- host -----------------------------------------------------------------------------

// How a call is cut.
struct SharedPlan {
  int rows, rt, zrows, part_rows, splits, least, own_blocks, own_least;
  long long units, segments, prefix_blocks;
  size_t prefix_o, prefix_ml, own_o, own_ml, places;
  size_t bytes() const { return prefix_o + prefix_ml + own_o + own_ml + places; }
  int ranges() const { return own_blocks * (kWaves / rt); }
};

constexpr size_t padded(size_t bytes) { return (bytes + 15) / 16 * 16; }

SharedPlan plan_of(const cudalm_paged_kv* kv, const cudalm_paged_query* q, const cudalm_paged_groups* g,
                   int new_tokens) {
  SharedPlan p;
  const int group = q->heads / kv->kv_heads, D = kv->head_dim, window = window_of(q);
  const long long B = kv->batch;
  p.rows = new_tokens * group;
  const int row_tiles = (p.rows + 15) / 16;
  p.rt = row_tiles > 2 ? 4 : row_tiles;
  p.zrows = (row_tiles + p.rt - 1) / p.rt;
  p.part_rows = 16 * p.rt < p.rows ? 16 * p.rt : p.rows;
  p.segments = B * kv->kv_heads * p.zrows;
  const int per_cu = D == 256 ? kPerCu<256> : D == 128 ? kPerCu<128> : kPerCu<64>, at_once = per_cu * cu_count();
  // What is expected: tiles of the longest prefix, and of all sequences' own tokens.
  const int len = expected_len(kv, q->max_len), prefix = expected_len(kv, g->max_shared);
  const long long near = window > 0 ? (window + sinks_of(q)) / kTile + 3LL : 1LL << 30;
  long long tiles = (prefix + kTile - 1) / kTile;
  tiles = tiles < near ? tiles : near;
  long long own = ((len > prefix ? len - prefix : len) + kTile - 1) / kTile + 1;
  own = p.segments * (own < near ? own : near);
  // Prefixes: a workgroup per `least` tiles. Fewer tiles end sooner but leave more parts, whose
  // bytes are written and read: t tiles cost t steps and all rows' parts 2 rows 4 D (tiles / t) at
  // 5 TB/s, least where the two are equal. And of the workgroups that run at once, one on every
  // CU is for own tokens (128 samples behind 32768 tokens, 256 channels: 70 us with half of them
  // for prefixes, 92 with two thirds; 5 documents, 128 channels: 39 and 35).
  const long long units = (B * p.rows + kRows - 1) / kRows * kv->kv_heads;
  const double bytes = 8.0 * B * p.rows * kv->kv_heads * D * tiles / 5e6, step = D == 256 ? 1.0 : D == 128 ? 0.8 : 0.6;
  long long least = static_cast<long long>(std::sqrt(bytes / step) + 0.5);
  const long long room = static_cast<long long>(per_cu - 1) * cu_count(), round = (units * tiles + room - 1) / room;
  least = least < round ? round : least;
  least = least < 1 ? 1 : least > tiles ? tiles : least;
  p.least = static_cast<int>(least);
  p.splits = static_cast<int>((tiles + least - 1) / least);
  p.units = B * p.rows / kRows + g->count;
  p.prefix_blocks = (static_cast<long long>(kv->kv_heads) * p.splits + 7) / 8 * 8 * p.units;
  const size_t blocks = static_cast<size_t>(p.splits) * p.units * kWaves * kv->kv_heads;
  p.prefix_o = blocks * 32 * D * 4;
  p.prefix_ml = blocks * 32 * 8;
  // Own tokens: what is left of a round of workgroups, a tile for a wave at least.
  long long most = at_once - units * p.splits;
  most = most > at_once / 4 ? most : at_once / 4;
  const long long need = (own * p.rt + kWaves - 1) / kWaves;
  p.own_blocks = static_cast<int>(need < most ? need : most);
  p.own_least = 1;
  const size_t slots = (2 * static_cast<size_t>(p.ranges()) + p.segments) * p.part_rows;
  p.own_o = slots * D * 4;
  p.own_ml = padded(slots * 8);
  p.places = static_cast<size_t>(p.segments) * 16;
  return p;
}

template <typename T, int D>
int launch(const SharedArgs& a, const SharedPlan& p, hipStream_t stream) {
  auto kernel = p.rt == 1 ? paged_shared_kernel<T, D, 1> : p.rt == 2 ? paged_shared_kernel<T, D, 2>
                                                                     : paged_shared_kernel<T, D, 4>;
  if (!allow_lds(kernel, kLdsBytes<D>)) return CUDALM_W4A16_ELAUNCH;
  const unsigned prefix = static_cast<unsigned>(p.prefix_blocks);
  kernel<<<prefix + p.own_blocks, 64 * kWaves, kLdsBytes<D>, stream>>>(a, prefix);
  if (const int rc = launch_status()) return rc;
  // Four pieces per wave read whole lines of rows; eight waves where there are parts for them;
  // where that makes few workgroups, more of both. (16 rows of 40 parts on 2 heads of 256: 5.2 us,
  // 6.0 with eight waves; 5120 rows of 128, 9 parts: 8.5, 10.2 with two pieces, 21 with sixteen
  // waves; 1024 rows of 256, 35 parts: 9.7, 10.2 with four waves, 13.6 with sixteen.)
  const long long parts = p.splits + p.ranges() / p.segments + 1;
  const unsigned tiles = static_cast<unsigned>((static_cast<long long>(a.kv.batch) * a.rows + 31) / 32) * a.kv.kv_heads;
  if (tiles * (D / 32) < static_cast<unsigned>(cu_count()) / 4)
    paged_shared_join_kernel<T, D, 2, 16><<<tiles * (D / 16), 1024, 0, stream>>>(a, D / 16);
  else if (parts > 16)
    paged_shared_join_kernel<T, D, 4, 8><<<tiles * (D / 32), 512, 0, stream>>>(a, D / 32);
  else
    paged_shared_join_kernel<T, D, 4, 4><<<tiles * (D / 32), 256, 0, stream>>>(a, D / 32);
  return launch_status();
}

template <typename T>
int launch_d(int D, const SharedArgs& a, const SharedPlan& p, hipStream_t stream) {
  return D == 64    ? launch<T, 64>(a, p, stream)
         : D == 128 ? launch<T, 128>(a, p, stream)
                    : launch<T, 256>(a, p, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, const cudalm_paged_groups* g, int new_tokens) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (!g) return CUDALM_W4A16_ENULL;
  if (new_tokens < 1 || g->count < 1 || g->count > kv->batch ||
      static_cast<long long>(new_tokens) * (q->heads / kv->kv_heads) > kMaxRows)
    return CUDALM_W4A16_EINVAL;
  if (!g->cu || !g->shared) return CUDALM_W4A16_ENULL;
  if (!aligned(g->cu, 4) || !aligned(g->shared, 4)) return CUDALM_W4A16_EALIGN;
  // rows, blocks of 32 of them and own tiles (with where the last range would end) are
  // numbered in 31 bits
  if (static_cast<long long>(kv->batch) * new_tokens * q->heads >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
  const SharedPlan p = plan_of(kv, q, g, new_tokens);
  const long long cap = (static_cast<long long>(kv->max_pages) * kv->page_size + kTile - 1) / kTile;
  const long long tiles = p.segments * (cap + 1), ranges = p.ranges();
  if (tiles + tiles / ranges + ranges >= (1LL << 31) || p.prefix_blocks + p.own_blocks >= kMaxGemmTiles ||
      p.units * kRows >= (1LL << 31))
    return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

}  // namespace
}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_paged_decode_shared_workspace_bytes(const cudalm_paged_kv* kv,
                                                             const cudalm_paged_query* q,
                                                             const cudalm_paged_groups* groups,
                                                             int new_tokens) {
  if (check(kv, q, groups, new_tokens) != CUDALM_W4A16_OK) return 0;
  return plan_of(kv, q, groups, new_tokens).bytes();
}

extern "C" int cudalm_paged_decode_shared(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                                          const cudalm_paged_groups* groups, int new_tokens,
                                          void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check(kv, q, groups, new_tokens)) return rc;
  if (!q->q || !q->out || !workspace) return CUDALM_W4A16_ENULL;
  if (!aligned(workspace, 16)) return CUDALM_W4A16_EALIGN;
  const SharedPlan p = plan_of(kv, q, groups, new_tokens);
  if (workspace_bytes < p.bytes()) return CUDALM_W4A16_ERANGE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t* at = ws;
    ws += bytes;
    return at;
  };
  SharedArgs a = {};
  a.kv = view_of(kv);
  a.sharing = {groups->cu, groups->shared, groups->count};
  a.k = static_cast<const uint16_t*>(kv->k);
  a.v = static_cast<const uint16_t*>(kv->v);
  a.q = static_cast<const uint16_t*>(q->q);
  a.out = static_cast<uint16_t*>(q->out);
  a.token_stride = q->token_stride;
  a.head_stride = q->head_stride;
  a.negate = q->scale < 0;
  // Not zero: hidden scores of -inf are multiplied by it.
  a.scale_log2 = fmaxf((a.negate ? -q->scale : q->scale) * kLog2e, 1e-38f);
  a.new_tokens = new_tokens;
  a.heads = q->heads;
  a.group = q->heads / kv->kv_heads;
  a.rows = p.rows;
  a.window = window_of(q);
  a.sinks = sinks_of(q);
  a.prefix_o = reinterpret_cast<f32x4_t*>(take(p.prefix_o));
  a.prefix_ml = reinterpret_cast<float2*>(take(p.prefix_ml));
  a.units = static_cast<int>(p.units);
  a.splits = p.splits;
  a.least = p.least;
  a.own_o = reinterpret_cast<float*>(take(p.own_o));
  a.own_ml = reinterpret_cast<float2*>(take(p.own_ml));
  a.places = reinterpret_cast<int4*>(take(p.places));
  a.zrows = p.zrows;
  a.part_rows = p.part_rows;
  a.ranges = p.ranges();
  a.own_least = p.own_least;
  return kv->type == CUDALM_PAGED_BF16 ? launch_d<PagedBf16>(kv->head_dim, a, p, stream)
                                       : launch_d<PagedF16>(kv->head_dim, a, p, stream);
}
