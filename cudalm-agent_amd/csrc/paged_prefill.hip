// Attention of a chunk of new tokens of every sequence over its pages, with a
// sliding window and sinks.
//
// The rows of a (sequence, key-value head) pair are its new tokens times the
// query heads of the group, so that a tile of rows covers few positions (little
// of it is above the diagonal) and a key or value is fetched once for the
// group. A wave holds 32 rows as the columns of 32x32x16 products:
//
//   S^T = K Q^T     (A = 32 tokens x 16 channels, B = 16 channels x 32 rows)
//   O^T += V^T P^T  (A = 32 channels x 16 tokens, B = 16 tokens x 32 rows)
//
// Q and O stay in registers. Tiles of keys and values go from the pages to LDS
// without passing registers, one tile ahead, for the waves of the workgroup.
// Row r of a tile of 32 keys in LDS is token r with bits 2 and 3 exchanged: then
// the eight scores that a lane holds of a row after the first product are
// those of eight consecutive tokens, which is its operand of the second. Key
// rows are stored with their 16-byte chunks exchanged by the row's low bits
// (chunk_exchange), or the lanes of a load, which read one chunk of many rows,
// would meet in the same banks; counters show no conflicts.
//
// The matrix and the vector unit bound it together: 32 tokens of 128 channels are 512
// cycles of products per wave, some 600 of exponentials, maxima and rounding, and the
// LDS reads of four waves fill 512 more. A chunk of 2048 tokens at 14336, 8 query heads on 2
// of 256: 233-257 us (card to card) and 15 for the join, 1.08 PFLOP/s at best, where an
// 8192-wide product of the library reaches 1.37. Two tiles of rows per wave halve the LDS
// reads but need more registers than two waves per SIMD leave (a 2048-token chunk at 6144,
// 32 heads on 8 of 128: 408 us, 261-288 with one). 8 prompts of up to 1000 tokens with a window
// of 512, same heads: 83-88 us, 19 tiles per workgroup of which 16 are the window's; 4% go
// into cleaning tiles that are seen in part.

#include <cstdint>

#include "paged_device.h"

namespace cudalm_hip {
namespace {

constexpr int kWaves = 4;           // of a workgroup, 32 rows each
constexpr int kRows = 32 * kWaves;
constexpr int kTile = 32;           // tokens per step
constexpr int kTileShift = 5;

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

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : D == 128 ? 3 : 4) void paged_prefill_kernel(const PrefillArgs a) {
  constexpr int KT = kTile, KK = D / 16, DT = D / 32;
  constexpr int C = D / 8;             // 16-byte chunks of a key row
  constexpr int kLoads = KT * D / 512; // 1 KB loads of a tile of keys (of values)
  constexpr int kTileElems = KT * D;
  extern __shared__ uint16_t lds[];    // [2][keys, values], then a vote per wave
  uint32_t* votes = reinterpret_cast<uint32_t*>(lds + 4 * kTileElems);
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 31, half = lane >> 5;

  const int hs = blockIdx.x % (a.kv.kv_heads * a.splits);
  const int unit = a.units - 1 - static_cast<int>(blockIdx.x) / (a.kv.kv_heads * a.splits);
  const int h = hs % a.kv.kv_heads, split = hs / a.kv.kv_heads;
  const int b = sequence_of(a.cu, a.kv.batch, unit, a.group, kRows, 1);
  if (b < 0) return;
  const int begin_row = load_uniform(a.cu + b), end_row = load_uniform(a.cu + b + 1);
  if (begin_row < 0 || end_row <= begin_row || end_row > a.tokens) return;
  const int new_tokens = end_row - begin_row;
  const int row0 = (unit - (begin_row * a.group / kRows + b)) * kRows;
  const int rows = new_tokens * a.group;
  if (row0 < 0 || row0 >= rows) return;  // (below 0 where cu does not ascend)
  const int length = a.kv.uniform_length(b), first = length - new_tokens;

  // this lane's row, and the positions of the wave's and the workgroup's first and last
  const int wave_row = row0 + 32 * wave, row = wave_row + n;
  const bool real = row < rows;
  const int j = (real ? row : rows - 1) / a.group;
  const int pos = real ? first + j : -1;
  const long long token = static_cast<long long>(begin_row) + j;
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
  auto position = [&](int row) { return first + (row < rows ? row : rows - 1) / a.group; };
  const int wave_first = position(wave_row), wave_last = position(wave_row + 31);
  const int wg_first = position(row0), wg_last = position(row0 + kRows - 1);
  const PagedTiles tiles(length, wg_first, wg_last, a.window, a.sinks, kTileShift);
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
    return t + KT - 1 <= from && (a.window <= 0 || t > to - a.window || t + KT - 1 < a.sinks);
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
      const int back = pos - t0 - 8 * half;
      const int sunk = t0 < a.sinks ? min(a.sinks - t0 - 8 * half, back + 1) : -1;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 16 * (e >> 3) + (e & 7);
        const bool sees = (static_cast<uint32_t>(back - i) < reach || i < sunk) &&
                          !((absent >> (e >> 3)) & 1);
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
            seen |= paged_sees(t + e, pos, a.window, a.sinks) ? 1u << e : 0u;
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

// One wave per (token, head): the join of the splits' partial sums. Bound by their bytes:
// 2048 tokens of 8 heads of 256 in four splits (75 MB): 15 us, 5 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(const PrefillArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long long rows = static_cast<long long>(a.tokens) * a.heads;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + wave_id();
  if (row >= rows) return;
  const int t = static_cast<int>(row / a.heads);
  if (t < load_uniform(a.cu) || t >= load_uniform(a.cu + a.kv.batch)) return;
  float M = kLowest;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_ml[2 * (s * rows + row)]);
  float acc[E] = {}, l = 0;
  for (int s = 0; s < a.splits; ++s) {
    const float ms = a.part_ml[2 * (s * rows + row)];
    if (ms == -__builtin_inff()) continue;
    const float w = exp2_fast(ms - M);
    l += w * a.part_ml[2 * (s * rows + row) + 1];
    const float* p = a.part_o + (s * rows + row) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += joined(w, p[e]);
  }
  float inv = 1.0f / l;
  if (l == 0.0f) {  // no weight at all: zeros, whatever the values
    inv = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0;
  }
  uint16_t* y = a.out + row * D + lane * E;
  if constexpr (E == 1) {
    y[0] = static_cast<uint16_t>(T::pack(acc[0] * inv, 0.0f));
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2)
      reinterpret_cast<uint32_t*>(y)[e / 2] = T::pack(acc[e] * inv, acc[e + 1] * inv);
  }
}

struct PrefillPlan {
  long long units;
  int splits, least;
  size_t o_bytes, ml_bytes;
  size_t bytes() const { return o_bytes + ml_bytes; }
};

PrefillPlan plan_of(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int tokens) {
  PrefillPlan p;
  const int group = q->heads / kv->kv_heads;
  p.units = static_cast<long long>(tokens) * group / kRows + kv->batch;
  const int len = expected_len(kv, q->max_len), window = window_of(q);
  long long tiles = (len + kTile - 1) / kTile;
  if (window > 0) {
    const long long near = (static_cast<long long>(window) + kRows / group + kTile) / kTile + 1 +
                           (sinks_of(q) + kTile - 1) / kTile;
    tiles = near < tiles ? near : tiles;
  }
  const long long groups = (static_cast<long long>(tokens) * group + kRows - 1) / kRows * kv->kv_heads;
  const long long most = tiles / 4;
  long long want = 2LL * cu_count() / groups;
  want = want < most ? want : most;
  want = want < 16 ? want : 16;
  p.splits = static_cast<int>(want < 1 ? 1 : want);
  p.least = 4;
  const size_t parts = static_cast<size_t>(p.splits) * tokens * q->heads;
  p.o_bytes = p.splits > 1 ? parts * kv->head_dim * 4 : 0;
  p.ml_bytes = p.splits > 1 ? parts * 8 : 0;
  return p;
}

template <typename T, int D>
int launch(const PrefillArgs& a, hipStream_t stream) {
  auto kernel = paged_prefill_kernel<T, D>;
  constexpr size_t kLds = 4 * kTile * D * 2 + 4 * kWaves;
  if (!allow_lds(kernel, kLds)) return CUDALM_W4A16_ELAUNCH;
  const unsigned grid = static_cast<unsigned>(a.units) * a.kv.kv_heads * a.splits;
  kernel<<<grid, 64 * kWaves, kLds, stream>>>(a);
  if (a.splits > 1) {
    if (const int rc = launch_status()) return rc;
    const long long rows = static_cast<long long>(a.tokens) * a.heads;
    paged_prefill_join_kernel<T, D><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(a);
  }
  return launch_status();
}

template <typename T>
int launch_d(int D, const PrefillArgs& a, hipStream_t stream) {
  return D == 64    ? launch<T, 64>(a, stream)
         : D == 128 ? launch<T, 128>(a, stream)
                    : launch<T, 256>(a, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int tokens) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (tokens < 0) return CUDALM_W4A16_EINVAL;
  const long long rows = static_cast<long long>(tokens) * q->heads;
  if (rows >= (1LL << 26)) return CUDALM_W4A16_ERANGE;
  if (tokens == 0) return CUDALM_W4A16_OK;
  const PrefillPlan p = plan_of(kv, q, tokens);
  if (p.units * kv->kv_heads * p.splits >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

template <typename T>
int regs_of_type(int D) {
  return D == 64    ? regs_of(paged_prefill_kernel<T, 64>)
         : D == 128 ? regs_of(paged_prefill_kernel<T, 128>)
                    : regs_of(paged_prefill_kernel<T, 256>);
}

}  // namespace

int paged_prefill_regs(int type, int D) {
  return type == CUDALM_PAGED_BF16 ? regs_of_type<PagedBf16>(D) : regs_of_type<PagedF16>(D);
}

}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_paged_prefill_workspace_bytes(const cudalm_paged_kv* kv,
                                                       const cudalm_paged_query* q, int tokens) {
  if (check(kv, q, tokens) != CUDALM_W4A16_OK || tokens == 0) return 0;
  return plan_of(kv, q, tokens).bytes();
}

extern "C" int cudalm_paged_prefill(const cudalm_paged_kv* kv, const cudalm_paged_query* q,
                                    const int32_t* cu_new, int tokens, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check(kv, q, tokens)) return rc;
  if (tokens == 0) return CUDALM_W4A16_OK;
  if (!q->q || !q->out || !cu_new) return CUDALM_W4A16_ENULL;
  if (!aligned(cu_new, 4)) return CUDALM_W4A16_EALIGN;
  const PrefillPlan p = plan_of(kv, q, tokens);
  if (p.bytes()) {
    if (!workspace) return CUDALM_W4A16_ENULL;
    if (!aligned(workspace, 16)) return CUDALM_W4A16_EALIGN;
    if (workspace_bytes < p.bytes()) return CUDALM_W4A16_ERANGE;
  }
  PrefillArgs a = {};
  a.kv = view_of(kv);
  a.k = static_cast<const uint16_t*>(kv->k);
  a.v = static_cast<const uint16_t*>(kv->v);
  a.q = static_cast<const uint16_t*>(q->q);
  a.out = static_cast<uint16_t*>(q->out);
  if (p.splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.o_bytes);
  }
  a.cu = cu_new;
  a.token_stride = q->token_stride;
  a.head_stride = q->head_stride;
  a.negate = q->scale < 0;
  // Not zero: hidden scores of -inf are multiplied by it.
  a.scale_log2 = fmaxf((a.negate ? -q->scale : q->scale) * kLog2e, 1e-38f);
  a.tokens = tokens;
  a.heads = q->heads;
  a.group = q->heads / kv->kv_heads;
  a.units = static_cast<int>(p.units);
  a.splits = p.splits;
  a.least = p.least;
  a.window = window_of(q);
  a.sinks = sinks_of(q);
  return kv->type == CUDALM_PAGED_BF16 ? launch_d<PagedBf16>(kv->head_dim, a, stream)
                                       : launch_d<PagedF16>(kv->head_dim, a, stream);
}
