// Attention of many rows of queries over one sequence's cached tokens: what prefill and
// decode with shared prefixes have in common (gfx950). How it works stands before
// prefill's kernel.
#ifndef CUDALM_PAGED_PREFILL_BODY_H
#define CUDALM_PAGED_PREFILL_BODY_H

#include <cstdint>
#include <type_traits>

#include "paged_shared.h"

namespace cudalm_hip {
namespace {

constexpr int kWaves = 4;           // of a workgroup, 32 rows each
constexpr int kRows = 32 * kWaves;

struct PrefillArgs {
  PagedView kv;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  uint16_t* out;
  float* part_o;   // [splits][tokens * heads][D], NULL: one split, straight to out
  float* part_ml;  // [splits][tokens * heads][2]
  const int32_t* cu;
  long long token_stride, head_stride;
  float scale_log2;
  int tokens, heads, group, units, splits, least, window, sinks;
  int negate;  // scale is negative: queries are negated and it is taken positive
};

// The rows of groups of sequences against their shared tokens: the group's sequences'
// `new_tokens` last tokens each, in a row, at positions of their own. In parts always.
struct PrefixArgs : PrefillArgs {
  SharedGroups sharing;
  int new_tokens;
};

// 16 bytes per lane from base (wave-uniform) + offset to LDS: lane i's land at
// dst + 16 i. Two loads at a time. The compiler's builtin for it makes every later
// LDS read wait for all such loads, the next tile's among them; here loads_landed()
// does the waiting.
__device__ __forceinline__ void load_lds16(const uint16_t* base0, uint32_t offset0, uint32_t dst0,
                                           const uint16_t* base1, uint32_t offset1, uint32_t dst1) {
  uint32_t saved;  // m0 holds the LDS address for the instruction
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\t"
      "s_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %6\n\ts_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(dst0), "v"(offset0), "s"(base0), "s"(dst1), "v"(offset1), "s"(base1)
      : "memory");
}

// This wave's loads to LDS have landed; a barrier after it speaks for all waves.
__device__ __forceinline__ void loads_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int swap_bits_2_3(int r) {
  return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
}

// Key row r has chunk c at place c ^ chunk_exchange(r): 16 rows of 64 channels lie in
// eight lines of 64 banks, two to a line, wider ones in one line or more each.
template <int D>
__device__ __forceinline__ int chunk_exchange(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}

// LDS of a workgroup.
template <int D>
constexpr size_t kPrefillLds = 4 * kTile * D * 2 + 4 * kWaves;

// Workgroup `block` of its call.
template <typename T, int D, typename Args>
__device__ __forceinline__ void paged_prefill_body(const Args& a, uint16_t* lds, unsigned block) {
  constexpr bool kPrefix = std::is_same<Args, PrefixArgs>::value;
  constexpr int KT = kTile, KK = D / 16, DT = D / 32;
  constexpr int C = D / 8;             // 16-byte chunks of a key row
  constexpr int kLoads = KT * D / 512; // 1 KB loads of a tile of keys (of values)
  constexpr int kTileElems = KT * D;
  // lds: [2][keys, values], then a vote per wave
  uint32_t* votes = reinterpret_cast<uint32_t*>(lds + 4 * kTileElems);
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 31, half = lane >> 5;

  const int hs = block % (a.kv.kv_heads * a.splits);
  const int unit = a.units - 1 - static_cast<int>(block) / (a.kv.kv_heads * a.splits);
  const int h = hs % a.kv.kv_heads, split = hs / a.kv.kv_heads;
  int b, begin_row, end_row;  // the sequence whose pages these are, and its rows of q
  if constexpr (kPrefix) {
    const int g = sequence_of(a.sharing.cu, a.sharing.count, unit, a.new_tokens * a.group, kRows, 1);
    int end;
    if (g < 0 || !a.sharing.sequences(g, a.kv.batch, &b, &end)) return;
    begin_row = b * a.new_tokens;
    end_row = end * a.new_tokens;
  } else {
    b = sequence_of(a.cu, a.kv.batch, unit, a.group, kRows, 1);
    if (b < 0) return;
    begin_row = load_uniform(a.cu + b);
    end_row = load_uniform(a.cu + b + 1);
    if (begin_row < 0 || end_row <= begin_row || end_row > a.tokens) return;
  }
  const int new_tokens = end_row - begin_row;
  int row0, length;
  if constexpr (kPrefix) {
    const int g = sequence_of(a.sharing.cu, a.sharing.count, unit, a.new_tokens * a.group, kRows, 1);
    row0 = (unit - (begin_row * a.group / kRows + g)) * kRows;
    length = a.sharing.tokens(a.kv, g);
  } else {
    row0 = (unit - (begin_row * a.group / kRows + b)) * kRows;
    length = a.kv.uniform_length(b);
  }
  const int rows = new_tokens * a.group;
  if (row0 < 0 || row0 >= rows) return;  // (below 0 where cu does not ascend)
  const int first = length - new_tokens;

  // this lane's row, and the positions of the wave's and the workgroup's first and last
  const int wave_row = row0 + 32 * wave, row = wave_row + n;
  const bool real = row < rows;
  const int j = (real ? row : rows - 1) / a.group;
  const long long token = static_cast<long long>(begin_row) + j;
  int pos = first + j;
  if constexpr (kPrefix) {
    const int s = static_cast<int>(token) / a.new_tokens;
    pos = a.kv.length(s) - a.new_tokens + static_cast<int>(token) - s * a.new_tokens;
  }
  const int row_pos = pos;  // (rows past the last stand for it)
  if (!real) pos = -1;
  const int head = h * a.group + (real ? row - j * a.group : 0);
  const long long out_row = token * a.heads + head;
  u32x4_t qf[KK];
  {
    const uint16_t* qp = a.q + token * a.token_stride + head * a.head_stride + 8 * half;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = *reinterpret_cast<const u32x4_t*>(qp + 16 * kk);
      if (a.negate) qf[kk] ^= 0x80008000u;
    }
  }
  int wave_first, wave_last, wg_first, wg_last;
  if constexpr (kPrefix) {
    wave_first = wave_last = row_pos;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      wave_first = min(wave_first, __shfl_xor(wave_first, x));
      wave_last = max(wave_last, __shfl_xor(wave_last, x));
    }
    wave_first = __builtin_amdgcn_readfirstlane(wave_first);
    wave_last = __builtin_amdgcn_readfirstlane(wave_last);
    int* seen = reinterpret_cast<int*>(lds);
    if (lane == 0) seen[2 * wave] = wave_first, seen[2 * wave + 1] = wave_last;
    __syncthreads();
    wg_first = seen[0], wg_last = seen[1];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) wg_first = min(wg_first, seen[2 * w]), wg_last = max(wg_last, seen[2 * w + 1]);
    wg_first = __builtin_amdgcn_readfirstlane(wg_first);
    wg_last = __builtin_amdgcn_readfirstlane(wg_last);
    __syncthreads();
  } else {
    auto position = [&](int row) { return first + (row < rows ? row : rows - 1) / a.group; };
    wave_first = position(wave_row), wave_last = position(wave_row + 31);
    wg_first = position(row0), wg_last = position(row0 + kRows - 1);
  }
  const auto tiles = [&] {
    if constexpr (kPrefix)
      return PagedRange(0, length, wg_first, wg_last, a.window, a.sinks, kTileShift);
    else
      return PagedTiles(length, wg_first, wg_last, a.window, a.sinks, kTileShift);
  }();
  const int per = tiles_per_split(tiles.count, a.splits, a.least);
  const int begin = split * per, end = begin + per < tiles.count ? begin + per : tiles.count;

  f32x16_t o[DT];
  float m = kLowest, l = 0;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = static_cast<size_t>(P) * D * a.kv.kv_heads;
  const size_t head_elems = static_cast<size_t>(P) * D * h;
  // A wave loads 1 KB pieces wave, wave + 4, .. of a tile's keys and values.
  // Key row r of piece 4 x + wave is r0 + x kStep: its token is that of r0 plus a number
  // that all lanes share, and the exchange of its chunks is the same for every x (but
  // for chunk bit 3 where D = 256). So one or two offsets per lane serve all loads.
  constexpr int kStep = 2048 / D;
  const int r0 = wave * (512 / D) + lane / C;
  const uint32_t k_lane =
      2 * (swap_bits_2_3(r0) % 16 * D + 8 * ((lane % C) ^ chunk_exchange<D>(r0)));
  const int v_piece = wave * 64;  // in channels of the tile's groups of eight tokens
  const uint32_t v_lane = 16 * (v_piece % D + lane);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + wave * 1024;

  // every row from position `from` to `to` sees all of the tile at t
  auto seen_whole = [&](int t, int from, int to) {
    return (!kPrefix || t + KT <= length) && t + KT - 1 <= from && (a.window <= 0 || t > to - a.window || t + KT - 1 < a.sinks);
  };
  const bool wg_full = row0 + kRows <= rows, wave_full = wave_row + 32 <= rows;
  // Places, pages and visibility of the next 32 tiles: lanes 2 i and 2 i + 1 hold the
  // halves of tile i, masks a bit each. One vector load of the table per 32 tiles,
  // and no scalar load in the loop.
  uint64_t half_at = 0;  // of the half's first key, and value, in its cache
  uint64_t absent_bits = 0, whole_bits = 0, wg_whole_bits = 0;
  int t0 = 0;
  auto look_ahead = [&](int i) {
    const int t = (tiles.tile(i + lane / 2) << kTileShift) + 16 * (lane & 1);
    int page = -1;
    if (i + lane / 2 < end) page = a.kv.page(b, t >> a.kv.page_shift);
    // absent pages are hidden below; any page will do
    half_at = max(page, 0) * page_elems + head_elems + static_cast<uint64_t>(t & (P - 1)) * D;
    absent_bits = __ballot(page < 0);
    const int first_token = t - 16 * (lane & 1);
    whole_bits = __ballot(wave_full && seen_whole(first_token, wave_first, wave_last));
    wg_whole_bits = __ballot(wg_full && seen_whole(first_token, wg_first, wg_last));
  };
  auto half_place = [&](int x) { return readlane64(half_at, x); };
  uint32_t absent = 0;  // of the tile fetched last: a bit for each half
  bool whole = false, wg_whole = false;
  auto fetch = [&](int i, int buf) {
    const int x = 2 * ((i - begin) & 31);
    if (x == 0) look_ahead(i);
    t0 = tiles.tile(i) << kTileShift;
    absent = static_cast<uint32_t>(absent_bits >> x) & 3;
    whole = !absent && ((whole_bits >> x) & 1);
    wg_whole = !absent && ((wg_whole_bits >> x) & 1);
    const uint64_t at0 = half_place(x), at1 = half_place(x + 1);
    const uint32_t kd = lds0 + buf * 4 * kTileElems, vd = kd + 2 * kTileElems;
#pragma unroll
    for (int y = 0; y < kLoads / kWaves; ++y) {
      // rows of the piece: tokens of 16-token half r / 16, bit 3 of r is bit 2 of the token
      const int r = y * kStep + wave * (512 / D), g = y * (2048 / (8 * D)) + v_piece / D;
      const bool odd = D == 256 && (y & 1);
      load_lds16(a.k + (r & 16 ? at1 : at0) + (odd ? 4 * D : 0), odd ? k_lane ^ 128 : k_lane,
                 kd + y * 4096, a.v + (g & 2 ? at1 : at0) + (g & 1) * 8 * D, v_lane, vd + y * 4096);
    }
  };
  // Zero weights times Inf or NaN are NaN. So in a tile that some row sees only
  // part of, values past the end or of absent pages (which may be anything) are
  // cleared, and Inf and NaN among the others taken out; the rows that do see
  // those get them at the end.
  uint32_t special = 0;
  auto clean = [&](u32x4_t* vt, int t0, uint32_t absent) {
#pragma unroll 2
    for (int u = threadIdx.x; u < KT / 8 * D; u += 64 * kWaves) {
      const int g = u / D, t = t0 + 8 * g;
      const bool gone = (absent >> (g >> 1)) & 1;
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

  // One tile of keys and values against the wave's rows.
  constexpr int kAhead = D == 256 ? 3 : 4;
  auto step = [&](bool whole, int t0, uint32_t absent, const uint16_t* kt, const uint16_t* vt) {
    __builtin_amdgcn_s_setprio(1);
    f32x16_t s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      s = T::mfma32(*reinterpret_cast<const u32x4_t*>(
                        kt + n * D + 8 * ((2 * kk + half) ^ chunk_exchange<D>(n))),
                    qf[kk], s);
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int kk = 0; kk < KK - kAhead; ++kk) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
    __builtin_amdgcn_s_setprio(0);
    // s[e] is the score of token t0 + 16 (e / 8) + 8 half + e % 8
    if (!whole) {
      // token t is seen from p if 0 <= p - t < window, or if t is a sink up to p
      const uint32_t reach = a.window > 0 ? a.window : 0x7FFFFFFF;
      const int back = pos - t0 - 8 * half, room = kPrefix ? length - t0 - 8 * half : 0;
      const int sunk = t0 < a.sinks ? min(a.sinks - t0 - 8 * half, back + 1) : -1;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 16 * (e >> 3) + (e & 7);
        const bool sees = (static_cast<uint32_t>(back - i) < reach || i < sunk) &&
                          !((absent >> (e >> 3)) & 1) && (!kPrefix || i < room);
        s[e] = sees ? s[e] : -__builtin_inff();
      }
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
    top = max_across_32(top) * a.scale_log2;
    // The maximum may lag by up to 2^8 (as in the decode kernel).
    if (__any(top > m + 8.0f)) {
      const float next = fmaxf(m, top), r = exp2_fast(m - next);
      l *= r;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= r;
      m = next;
    }
    u32x4_t pf[2];
    float sum = 0;
    const u32x4_t* vp = reinterpret_cast<const u32x4_t*>(vt) + half * D + n;
    constexpr int kFirst = 1 + D / 128;  // value operands that load during the exponentials
    u32x4_t vf[kFirst];
#pragma unroll
    for (int x = 0; x < kFirst; ++x) vf[x] = vp[(x / DT) * 2 * D + 32 * (x % DT)];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float p0 = exp2_fast(__builtin_fmaf(s[e], a.scale_log2, -m));
      const float p1 = exp2_fast(__builtin_fmaf(s[e + 1], a.scale_log2, -m));
      sum += p0 + p1;
      // rounded to the values' type, as the matrix unit takes them
      pf[e / 8][e % 8 / 2] = T::pack(p0, p1);
    }
    l += sum;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < 2 * DT; ++x) {
      const u32x4_t w = vf[x % kFirst];
      if (x + kFirst < 2 * DT) vf[x % kFirst] = vp[((x + kFirst) / DT) * 2 * D + 32 * ((x + kFirst) % DT)];
      o[x % DT] = T::mfma32(w, pf[x / DT], o[x % DT]);
    }
    if (D >= 128) {
      __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
      for (int x = 0; x < 2 * DT - kFirst; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kFirst, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0;
  int buf = 0;
  if (begin < end) fetch(begin, 0);
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    uint16_t* kt = lds + buf * 2 * kTileElems;
    uint16_t* vt = kt + kTileElems;
    const int here = t0;
    const uint32_t gone = absent;
    const bool seen = whole, wg_seen = wg_whole;
    loads_landed();
    __syncthreads();  // this tile has landed for all waves; the other buffer is free
    buf ^= 1;
    if (i + 1 < end) fetch(i + 1, buf);
    if (!wg_seen) {
      clean(reinterpret_cast<u32x4_t*>(vt), here, gone);
      __syncthreads();
    }
    if (here <= wave_last) step(seen, here, gone, kt, vt);  // not above the wave's rows
  }
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
            seen |= paged_sees(t + e, pos, a.window, a.sinks) && (!kPrefix || t + e < length) ? 1u << e : 0u;
          w = *reinterpret_cast<const u32x4_t*>(a.v + page * page_elems + head_elems +
                                                static_cast<size_t>(t & (P - 1)) * D +
                                                8 * (32 * dt + n));
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
  votes[wave] = __any(special != 0 || !(most[0] < __builtin_inff()));
  __syncthreads();
  special = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) special |= votes[w];
  special = __builtin_amdgcn_readfirstlane(special);
  l += __shfl_xor(l, 32);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const size_t at = static_cast<size_t>(split) * a.tokens * a.heads + out_row;
  // -inf tells the join that there is nothing to read: no weight here, nor Inf or NaN
  if (a.part_o && real && half == 0) {
    a.part_ml[2 * at] = l == 0.0f && !special ? -__builtin_inff() : m;
    a.part_ml[2 * at + 1] = l;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    f32x16_t r = o[dt];
    if (special) {
      add_special(r, dt);
      // (no weight at all: zeros, whatever the values; parts keep theirs for the join)
      if (l == 0.0f && !a.part_o) r = 0.0f;
    }
    if (!real) continue;
    if (a.part_o) {
      if (begin >= end) continue;  // (l is zero)
      float* p = a.part_o + at * D + 32 * dt + 4 * half;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        *reinterpret_cast<f32x4_t*>(p + 8 * y) =
            f32x4_t{r[4 * y], r[4 * y + 1], r[4 * y + 2], r[4 * y + 3]};
    } else {
      uint16_t* out = a.out + out_row * D + 32 * dt + 4 * half;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        *reinterpret_cast<u32x2_t*>(out + 8 * y) =
            u32x2_t{T::pack(r[4 * y] * inv, r[4 * y + 1] * inv),
                    T::pack(r[4 * y + 2] * inv, r[4 * y + 3] * inv)};
    }
  }
}

}  // namespace
}  // namespace cudalm_hip

#endif
