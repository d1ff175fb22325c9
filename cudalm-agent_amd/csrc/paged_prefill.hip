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
// (chunk c at c ^ (r & 7)), or the lanes of a load, which read one chunk of
// many rows, would meet in the same banks.

#include <cstdint>
#include <type_traits>

#include "paged_device.h"

namespace cudalm_hip {
namespace {

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
};

// 16 bytes per lane from memory to LDS: lane i's land at dst + 16 i. The
// compiler's builtin for it makes every later LDS read wait for all such loads,
// the next tile's among them; here loads_landed() does the waiting.
__device__ __forceinline__ void load_lds16(const uint16_t* src, uint16_t* dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>(dst)));
  uint32_t saved;  // m0 holds the LDS address for the instruction
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(at), "v"(src)
      : "memory");
}

// This wave's loads to LDS have landed; a barrier after it speaks for all waves.
__device__ __forceinline__ void loads_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int swap_bits_2_3(int r) {
  return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
}

template <typename T, int D, int NW, int KT>
__global__ __launch_bounds__(64 * NW, 2) void paged_prefill_kernel(const PrefillArgs a) {
  constexpr int kShift = KT == 64 ? 6 : 5;
  constexpr int KK = D / 16, DT = D / 32, ST = KT / 32;
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
  const int b = sequence_of(a.cu, a.kv.batch, unit, a.group, 32 * NW, 1);
  if (b < 0) return;
  const int begin_row = load_uniform(a.cu + b), new_tokens = load_uniform(a.cu + b + 1) - begin_row;
  if (begin_row < 0 || new_tokens < 1 || begin_row + new_tokens > a.tokens) return;
  const int row0 = (unit - (begin_row * a.group / (32 * NW) + b)) * 32 * NW;
  const int rows = new_tokens * a.group;
  if (row0 >= rows) return;
  const int length = a.kv.uniform_length(b), first = length - new_tokens;

  // this lane's row, and the positions of the workgroup's first and last
  const int row = row0 + wave * 32 + n;
  const bool real = row < rows;
  const int j = (real ? row : rows - 1) / a.group;
  const int pos = real ? first + j : -1;
  const int wg_first = first + row0 / a.group;
  const int wg_last = first + (row0 + 32 * NW - 1 < rows ? row0 + 32 * NW - 1 : rows - 1) / a.group;
  const PagedTiles tiles(length, wg_first, wg_last, a.window, a.sinks, kShift);
  const int per = tiles_per_split(tiles.count, a.splits, a.least, 1);
  const int begin = split * per, end = begin + per < tiles.count ? begin + per : tiles.count;

  const long long token = static_cast<long long>(begin_row) + j;
  const int head = h * a.group + (real ? row - j * a.group : 0);
  const long long out_row = token * a.heads + head;

  u32x4_t qf[KK];
  {
    const uint16_t* qp = a.q + token * a.token_stride + head * a.head_stride + 8 * half;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = *reinterpret_cast<const u32x4_t*>(qp + 16 * kk);
  }
  f32x16_t o[DT];
  float m = kLowest, l = 0;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = static_cast<size_t>(P) * D * a.kv.kv_heads;
  const size_t head_elems = static_cast<size_t>(P) * D * h;
  // what this lane loads of a 1 KB piece of keys: row and chunk
  const int piece_row = lane / C, piece_slot = lane % C;

  // A tile's pages, and whether every row of the workgroup sees all of it.
  int t0 = 0, page0 = -1, page1 = -1, page2 = -1, page3 = -1;  // of 16 tokens each
  auto look_up = [&](int i) {
    t0 = tiles.tile(i) << kShift;
    const int s = a.kv.page_shift;
    page0 = a.kv.uniform_page(b, t0 >> s);
    page1 = a.kv.uniform_page(b, (t0 + 16) >> s);
    page2 = KT > 32 ? a.kv.uniform_page(b, (t0 + 32) >> s) : page0;
    page3 = KT > 32 ? a.kv.uniform_page(b, (t0 + 48) >> s) : page0;
    return page0 >= 0 && page1 >= 0 && page2 >= 0 && page3 >= 0 && t0 + KT - 1 <= wg_first && row0 + 32 * NW <= rows &&
           (a.window <= 0 || t0 > wg_last - a.window || t0 + KT - 1 < a.sinks);
  };
  auto fetch = [&](int buf) {
    // absent pages are hidden below; any page will do
    const int g0 = max(page0, 0), g1 = max(page1, 0), g2 = max(page2, 0), g3 = max(page3, 0);
    uint16_t* kd = lds + buf * 2 * kTileElems;
    uint16_t* vd = kd + kTileElems;
#pragma unroll
    for (int x = 0; x < kLoads / NW; ++x) {
      const int piece = x * NW + wave;
      {
        const int r = piece * (64 / C) + piece_row;
        const int tok = swap_bits_2_3(r);
        // (rows of a piece are tokens of the same 16)
        const int x16 = (piece * (64 / C)) >> 4;
        const int pg = x16 < 2 ? (x16 ? g1 : g0) : x16 == 2 ? g2 : g3;
        const uint16_t* src = a.k + pg * page_elems + head_elems +
                              static_cast<size_t>((t0 + tok) & (P - 1)) * D +
                              8 * (piece_slot ^ (r & 7));
        load_lds16(src, kd + piece * 512);
      }
      {
        const int g = piece * 64 / D;  // group of eight tokens
        const int x16 = g >> 1;
        const int pg = x16 < 2 ? (x16 ? g1 : g0) : x16 == 2 ? g2 : g3;
        const uint16_t* src = a.v + pg * page_elems + head_elems +
                              static_cast<size_t>((t0 + 8 * g) & (P - 1)) * D +
                              8 * (piece * 64 % D + lane);
        load_lds16(src, vd + piece * 512);
      }
    }
  };

#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0;
  // One tile of keys and values against the wave's rows.
  uint32_t seen[ST];  // which of a lane's 16 scores (of 32 tokens) its row sees
  auto step = [&](auto masked, const uint16_t* kt, const uint16_t* vt) {
    constexpr bool kMasked = decltype(masked)::value;
    f32x16_t s[ST];
#pragma unroll
    for (int st = 0; st < ST; ++st) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[st][e] = 0;
      const int r = 32 * st + n;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(
            kt + r * D + 8 * ((2 * kk + half) ^ (r & 7)));
        s[st] = T::mfma32(kf, qf[kk], s[st]);
      }
    }
#pragma unroll
    for (int st = 0; st < ST; ++st) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[st][e] *= a.scale_log2;
        if (kMasked) s[st][e] = (seen[st] >> e) & 1 ? s[st][e] : -__builtin_inff();
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[st][e]);
    top = fmaxf(top, __shfl_xor(top, 32));
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
    u32x4_t pf[2 * ST];
    float sum = 0;
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = exp2_fast(s[st][e] - m), p1 = exp2_fast(s[st][e + 1] - m);
        sum += p0 + p1;
        // rounded to the values' type, as the matrix unit takes them
        pf[2 * st + e / 8][e % 8 / 2] = T::pack(p0, p1);
      }
    l += sum;
#pragma unroll
    for (int x = 0; x < 2 * ST; ++x)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4_t vf =
            *reinterpret_cast<const u32x4_t*>(vt + ((2 * x + half) * D + 32 * dt + n) * 8);
        o[dt] = T::mfma32(vf, pf[x], o[dt]);
      }
  };

  // Tiles that every row sees whole, the next one on its way meanwhile.
  int i = begin, buf = 0;
  while (i < end && !look_up(i)) ++i;
  if (i < end) fetch(0);
  while (i < end) {
    loads_landed();
    __syncthreads();  // this tile has landed for all waves; the other buffer is free
    do ++i;
    while (i < end && !look_up(i));
    if (i < end) fetch(buf ^ 1);
    step(std::false_type{}, lds + buf * 2 * kTileElems, lds + (buf * 2 + 1) * kTileElems);
    buf ^= 1;
  }
  // The others: at the diagonal, the ends of the window and the sinks, and
  // where pages are absent.
#pragma unroll 1
  for (i = begin; i < end; ++i) {
    if (look_up(i)) continue;
    __syncthreads();
    fetch(0);
    const uint32_t absent = (page0 < 0) | (page1 < 0) << 1 | (page2 < 0) << 2 | (page3 < 0) << 3;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      seen[st] = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int t = 32 * st + 16 * (e >> 3) + 8 * half + (e & 7);
        seen[st] |= paged_sees(t0 + t, pos, a.window, a.sinks) ? 1u << e : 0u;
      }
      const uint32_t gone = absent >> (2 * st);
      seen[st] &= ~((gone & 1 ? 0x00FFu : 0u) | (gone & 2 ? 0xFF00u : 0u));
    }
    loads_landed();
    __syncthreads();
    // Values that no row sees may be anything: clear them. Look whether the
    // others are finite.
    u32x4_t* vt = reinterpret_cast<u32x4_t*>(lds + kTileElems);
    uint32_t special = 0;
    for (int u = threadIdx.x; u < KT / 8 * D; u += 64 * NW) {
      const int g = u / D, t = t0 + 8 * g;
      u32x4_t w = vt[u];
      const bool gone = (absent >> (g >> 1)) & 1;
      if (gone || t + 8 > length) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (gone || t + 2 * e >= length) w[e] &= 0xFFFF0000u;
          if (gone || t + 2 * e + 1 >= length) w[e] &= 0x0000FFFFu;
        }
        vt[u] = w;
      }
      special |= special_bits<T>(w);
    }
    if (lane == 0) votes[wave] = 0;
    if (__any(special != 0) && lane == 0) votes[wave] = 1;
    __syncthreads();
    special = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) special |= votes[w];
    if (special) {
      for (int u = threadIdx.x; u < KT / 8 * D; u += 64 * NW) vt[u] = finite_part<T>(vt[u]);
      __syncthreads();
    }
    step(std::true_type{}, lds, lds + kTileElems);
    if (special) {
      __syncthreads();
      fetch(0);
      loads_landed();
      __syncthreads();
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int flip = 0; flip < 2; ++flip) {
          f32x16_t count;
#pragma unroll
          for (int e = 0; e < 16; ++e) count[e] = 0;
#pragma unroll
          for (int x = 0; x < 2 * ST; ++x)
            count = T::mfma32(special_part<T>(vt[(2 * x + half) * D + 32 * dt + n], flip - 1),
                              seen_operand<T>(seen[x / 2] >> (8 * (x & 1))), count);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[dt][e] += count[e] > 0 ? (flip ? -__builtin_inff() : __builtin_inff()) : 0.0f;
          asm volatile("" ::: "memory");  // one at a time: few registers over speed here
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  l += __shfl_xor(l, 32);
  if (!real) return;
  if (a.part_o) {
    const size_t at = static_cast<size_t>(split) * a.tokens * a.heads + out_row;
    if (half == 0) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
    if (begin >= end) return;
    float* p = a.part_o + at * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f32x4_t*>(p + 32 * dt + 8 * x) =
            f32x4_t{o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* y = a.out + out_row * D + 4 * half;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<u32x2_t*>(y + 32 * dt + 8 * x) =
          u32x2_t{T::pack(o[dt][4 * x] * inv, o[dt][4 * x + 1] * inv),
                  T::pack(o[dt][4 * x + 2] * inv, o[dt][4 * x + 3] * inv)};
}

// One wave per (token, head): the join of the splits' partial sums.
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
    const float ls = a.part_ml[2 * (s * rows + row) + 1];
    if (ls == 0.0f) continue;  // no tokens: nothing was written
    const float w = exp2_fast(a.part_ml[2 * (s * rows + row)] - M);
    l += w * ls;
    const float* p = a.part_o + (s * rows + row) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += w * p[e];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* y = a.out + row * D + lane * E;
  if constexpr (E == 1) {
    y[0] = static_cast<uint16_t>(T::pack(acc[0] * inv, 0.0f));
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2)
      reinterpret_cast<uint32_t*>(y)[e / 2] = T::pack(acc[e] * inv, acc[e + 1] * inv);
  }
}

constexpr int kWaves = 4;

template <int D>
constexpr int tile_tokens() {
  return D == 256 ? 32 : 64;
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
  const int kt = kv->head_dim == 256 ? 32 : 64;
  p.units = static_cast<long long>(tokens) * group / (32 * kWaves) + kv->batch;
  const int len = expected_len(kv, q->max_len), window = window_of(q);
  long long tiles = (len + kt - 1) / kt;
  if (window > 0) {
    const long long near = (static_cast<long long>(window) + 32 * kWaves / group + kt) / kt + 1 +
                           (sinks_of(q) + kt - 1) / kt;
    tiles = near < tiles ? near : tiles;
  }
  const long long groups = p.units * kv->kv_heads;
  long long want = 2LL * cu_count() / groups;
  const long long most = tiles / 4;
  want = want < most ? want : most;
  want = want < 16 ? want : 16;
  p.splits = static_cast<int>(want < 1 ? 1 : want);
  p.least = static_cast<int>((tiles + p.splits - 1) / p.splits);
  if (p.least < 1) p.least = 1;
  // a shorter range of tiles (rows early in a chunk) still uses all splits
  p.least = p.least < 4 ? p.least : 4;
  const size_t parts = static_cast<size_t>(p.splits) * tokens * q->heads;
  p.o_bytes = p.splits > 1 ? parts * kv->head_dim * 4 : 0;
  p.ml_bytes = p.splits > 1 ? parts * 8 : 0;
  return p;
}

template <typename T, int D>
int launch(const PrefillArgs& a, hipStream_t stream) {
  constexpr int KT = tile_tokens<D>();
  auto kernel = paged_prefill_kernel<T, D, kWaves, KT>;
  constexpr size_t kLds = 4 * KT * D * 2 + 4 * kWaves;
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
  return D == 64 ? launch<T, 64>(a, stream) : D == 128 ? launch<T, 128>(a, stream) : launch<T, 256>(a, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int tokens) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (tokens < 0) return CUDALM_W4A16_EINVAL;
  const long long rows = static_cast<long long>(tokens) * q->heads;
  if (rows >= (1LL << 26)) return CUDALM_W4A16_ERANGE;
  const PrefillPlan p = plan_of(kv, q, tokens);
  if (p.units * kv->kv_heads * p.splits >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

template <typename T>
int regs_of_type(int D) {
  return D == 64    ? regs_of(paged_prefill_kernel<T, 64, kWaves, tile_tokens<64>()>)
         : D == 128 ? regs_of(paged_prefill_kernel<T, 128, kWaves, tile_tokens<128>()>)
                    : regs_of(paged_prefill_kernel<T, 256, kWaves, tile_tokens<256>()>);
}

}  // namespace

int paged_prefill_regs(int type, int D) {
  return type == CUDALM_PAGED_BF16 ? regs_of_type<PagedBf16>(D) : regs_of_type<PagedF16>(D);
}

}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_paged_prefill_workspace_bytes(const cudalm_paged_kv* kv,
                                                       const cudalm_paged_query* q, int tokens) {
  if (check(kv, q, tokens) != CUDALM_W4A16_OK) return 0;
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
  a.scale_log2 = q->scale * kLog2e;
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
