// Low-rank adapters of many requests beside shared projections: two products with a
// rank between them, h = A x and y + s B h, over tiles of up to 16 rows that have the
// same adapter.
//
// Rows are the columns of the matrix products (16x16x32), so that an adapter's factors
// are read as they lie, 16 bytes of a row per lane, and one tile reads them once for
// its rows. h is summed in fp32 over the waves of a workgroup. The second product takes
// bf16 operands only: h = hh + hl, two bf16 numbers, keep 16 of its bits and all of fp32's
// range, which fp16 would not; fp16 factors are split in the same way, b = bh + bl, exactly.
// h is therefore stored as sections of `rank` numbers each along the summed index,
//
//   h:  hh | hl            (fp16: hh | hl | hh without Inf and NaN)
//   b:  b  | b without Inf and NaN          (fp16: bh | bh without .. | bl)
//
// so that the products of a section meet and Inf times 0 comes up only where the
// unsplit factors have it.

#include "cudalm_lora.h"

#include "paged_device.h"

namespace cudalm_hip {
namespace {

constexpr int kRows = 16;        // of a tile
constexpr int kPlanThreads = 1024;

// A plan: the number of tiles, three words, the tiles, and the rows in their order.
struct LoraTile {
  int adapter, start, count, unused;  // adapter -1: rows of none
};
struct LoraPlan {
  int tiles, unused[3];
};

int most_tiles(int M, int adapters) {
  const int groups = adapters < M ? adapters + 1 : M;  // and the rows of none
  const long long n = (static_cast<long long>(M) + kRows - 1) / kRows + groups;
  return n < M ? static_cast<int>(n) : M;
}

struct PlanArgs {
  const int32_t* index;
  LoraPlan* plan;
  LoraTile* tiles;
  int32_t* order;
  int M, adapters;
};

// For every lane with a number a (a < 0: none): how much counter[a] was before the lanes
// up to this one added one each, those of a wave in their order.
__device__ __forceinline__ int claim(int* counter, int a) {
  int at = 0;
  const int lane = threadIdx.x & 63;
  uint64_t left = __ballot(a >= 0);
  while (left) {
    const int leader = __builtin_ctzll(left);
    const int one = __builtin_amdgcn_readlane(a, leader);
    const uint64_t same = __ballot(a == one);
    int base = 0;
    if (lane == leader) base = atomicAdd(&counter[one], static_cast<int>(__popcll(same)));
    base = __builtin_amdgcn_readlane(base, leader);
    if (a == one) at = base + static_cast<int>(__popcll(same & ((1ULL << lane) - 1)));
    left &= ~same;
  }
  return at;
}

// One workgroup: rows per adapter, where each adapter's begin, its tiles, its rows. Which
// of two waves adds its rows first is open; no result depends on it, since every row is
// a column of its own in the products.
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const PlanArgs a) {
  extern __shared__ int counter[];  // [adapters + 1], the last for rows of none
  __shared__ int rows_of[kPlanThreads / 64], tiles_of[kPlanThreads / 64];
  const int groups = a.adapters + 1, lane = threadIdx.x & 63, wave = wave_id();
  for (int i = threadIdx.x; i < groups; i += kPlanThreads) counter[i] = 0;
  __syncthreads();
  auto group_of = [&](int m) {
    const int i = a.index[m];
    return i >= 0 && i < a.adapters ? i : a.adapters;
  };
  for (int m0 = 64 * wave; m0 < a.M; m0 += kPlanThreads)
    claim(counter, m0 + lane < a.M ? group_of(m0 + lane) : -1);
  __syncthreads();
  // running sums over the groups, a stretch of them per thread
  const int each = (groups + kPlanThreads - 1) / kPlanThreads;
  const int from = threadIdx.x * each, to = from + each < groups ? from + each : groups;
  int rows = 0, tiles = 0;
  for (int i = from; i < to; ++i) rows += counter[i], tiles += (counter[i] + kRows - 1) / kRows;
  int rows_before = rows, tiles_before = tiles;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const int r = __shfl_up(rows_before, x), t = __shfl_up(tiles_before, x);
    if (lane >= x) rows_before += r, tiles_before += t;
  }
  if (lane == 63) rows_of[wave] = rows_before, tiles_of[wave] = tiles_before;
  __syncthreads();
  rows_before -= rows;
  tiles_before -= tiles;
  for (int w = 0; w < wave; ++w) rows_before += rows_of[w], tiles_before += tiles_of[w];
  if (threadIdx.x == kPlanThreads - 1) a.plan->tiles = tiles_before + tiles;
  for (int i = from; i < to; ++i) {
    const int n = counter[i];
    counter[i] = rows_before;
    for (int r = 0; r < n; r += kRows)
      a.tiles[tiles_before++] = {i < a.adapters ? i : -1, rows_before + r, n - r < kRows ? n - r : kRows, 0};
    rows_before += n;
  }
  __syncthreads();
  for (int m0 = 64 * wave; m0 < a.M; m0 += kPlanThreads) {
    const int m = m0 + lane;
    const int at = claim(counter, m < a.M ? group_of(m) : -1);
    if (m < a.M) a.order[at] = m;
  }
}

struct ShrinkArgs {
  const LoraPlan* plan;
  const LoraTile* tiles;
  const int32_t* order;
  const int32_t* ranks;  // or NULL
  const uint16_t* x;
  uint16_t* h;  // [projection][M][sections * rank]
  const uint16_t* a[CUDALM_LORA_MAX_PROJ];
  long long x_stride;
  int K, M, rank, rank_tiles, total;  // rank_tiles: of a projection; total: of all
};

struct ExpandArgs {
  const LoraPlan* plan;
  const LoraTile* tiles;
  const int32_t* order;
  const int32_t* ranks;
  const float* scales;  // or NULL
  const uint16_t* h;
  const uint16_t* b[CUDALM_LORA_MAX_PROJ];
  const uint16_t* y[CUDALM_LORA_MAX_PROJ];
  uint16_t* out[CUDALM_LORA_MAX_PROJ];
  long long y_stride[CUDALM_LORA_MAX_PROJ], out_stride[CUDALM_LORA_MAX_PROJ];
  int N[CUDALM_LORA_MAX_PROJ], chunk0[CUDALM_LORA_MAX_PROJ];  // first chunk of columns of each
  int count, M, rank, wide;  // wide: a bit for each projection whose rows go 16 bytes at a time
};

template <typename T>
constexpr int kSections = T::kExp == PagedBf16::kExp ? 2 : 3;

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < __builtin_inff() ? x : 0.0f; }

// A number as bf16 and the rest of it, which is 0 beside Inf and NaN.
__device__ __forceinline__ void split(float x, float& hi, float& lo) {
  hi = bf16_lo(f32_to_bf16_rne(x));
  lo = finite_or_zero(x - hi);
}

// h of one tile and RT x 16 ranks: the waves split K.
template <typename T, int RT, int WV>
__global__ __launch_bounds__(64 * WV) void lora_shrink_kernel(const ShrinkArgs a) {
  constexpr int kSec = kSections<T>;
  __shared__ float sums[WV][RT][256];
  const int groups = (a.total + RT - 1) / RT;
  const int t = blockIdx.x / groups, rt0 = blockIdx.x % groups * RT;
  if (t >= load_uniform(&a.plan->tiles)) return;
  const int adapter = load_uniform(&a.tiles[t].adapter);
  if (adapter < 0) return;
  const int start = load_uniform(&a.tiles[t].start), count = load_uniform(&a.tiles[t].count);
  const int rank = a.ranks ? load_uniform(a.ranks + adapter) : a.rank;
  const int lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15, quarter = lane >> 4;
  const uint16_t* x = a.x + a.order[start + (n < count ? n : 0)] * a.x_stride + 8 * quarter;
  const uint16_t* factor[RT];
  bool real[RT];
  f32x4_t sum[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int rt = rt0 + i, p = rt / a.rank_tiles, r = rt % a.rank_tiles * 16 + n;
    real[i] = rt < a.total && r < rank && r < a.rank;
    factor[i] = a.a[rt < a.total ? p : 0] +
                (static_cast<size_t>(adapter) * a.rank + (real[i] ? r : 0)) * a.K + 8 * quarter;
    sum[i] = f32x4_t{0, 0, 0, 0};
  }
#pragma unroll 4
  for (int k = 32 * wave; k < a.K; k += 32 * WV) {
    const bool in = k + 8 * quarter < a.K;
    const u32x4_t none = {0, 0, 0, 0};
    const u32x4_t xf = in ? load16(x + k) : none;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const u32x4_t af = in && real[i] ? load16(factor[i] + k) : none;
      sum[i] = T::mfma(af, xf, sum[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)  // rank 4 quarter + e of row n
    *reinterpret_cast<f32x4_t*>(&sums[wave][i][16 * n + 4 * quarter]) = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < RT * 256; i += 64 * WV) {
    const int rt = rt0 + i / 256, r = rt % a.rank_tiles * 16 + i % 16, m = i / 16 % 16;
    if (rt >= a.total || r >= a.rank || m >= count) continue;
    float v = 0, hi, lo;
#pragma unroll
    for (int w = 0; w < WV; ++w) v += sums[w][i / 256][i % 256];
    split(v, hi, lo);
    uint16_t* h = a.h + (static_cast<size_t>(rt / a.rank_tiles) * a.M + start + m) * (kSec * a.rank) + r;
    h[0] = static_cast<uint16_t>(f32_to_bf16_rne(hi));
    h[a.rank] = static_cast<uint16_t>(f32_to_bf16_rne(lo));
    if (kSec == 3) h[2 * a.rank] = static_cast<uint16_t>(f32_to_bf16_rne(finite_or_zero(hi)));
  }
}

// Eight factors as section `sec` of the second product takes them.
template <typename T>
__device__ __forceinline__ u32x4_t section_of(u32x4_t b, int sec) {
  if constexpr (kSections<T> == 2) {
    return sec ? finite_part<PagedBf16>(b) : b;
  } else {
    u32x4_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float h0, l0, h1, l1;
      split(T::value(static_cast<uint16_t>(b[e])), h0, l0);
      split(T::value(static_cast<uint16_t>(b[e] >> 16)), h1, l1);
      r[e] = sec == 2 ? f32_to_bf16_rne2(l0, l1) : f32_to_bf16_rne2(h0, h1);
    }
    return sec == 1 ? finite_part<PagedBf16>(r) : r;
  }
}

// 32 columns of TG tiles of rows per wave and step, `steps` of them: lane (n, quarter)
// holds columns 8 quarter .. + 7 of row n, from two products whose rows stand for columns 8 (i / 4) +
// 4 f + i % 4.
template <typename T, int TG, int WV>
__global__ __launch_bounds__(64 * WV) void lora_expand_kernel(const ExpandArgs a, int chunks, int steps) {
  constexpr int kSec = kSections<T>;
  const int group = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int tiles = load_uniform(&a.plan->tiles);
  if (group * TG >= tiles) return;
  int p = 0;
  while (p + 1 < a.count && chunk >= a.chunk0[p + 1]) ++p;
  const int lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15, quarter = lane >> 4;
  const int N = a.N[p];
  const bool wide = (a.wide >> p) & 1;
  const uint16_t* y = a.y[p];
  uint16_t* out = a.out[p];
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    const int n0 = ((chunk - a.chunk0[p]) * steps + step) * 32 * WV + 32 * wave;
    if (n0 >= N) break;
    const int col = n0 + 8 * quarter;
    const int row_a = n0 + 8 * (n >> 2) + (n & 3);  // and 4 further
#pragma unroll 1
    for (int t = group * TG; t < tiles && t < (group + 1) * TG; ++t) {
      const int adapter = load_uniform(&a.tiles[t].adapter);
      const int start = load_uniform(&a.tiles[t].start), count = load_uniform(&a.tiles[t].count);
      if (adapter < 0 && y == out) continue;
      const int m = a.order[start + (n < count ? n : 0)];
      f32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
      float scale = 0;
      if (adapter >= 0) {
        const int rank = min(a.rank, a.ranks ? load_uniform(a.ranks + adapter) : a.rank);
        scale = a.scales ? a.scales[adapter] : 1.0f;
        const uint16_t* h = a.h + (static_cast<size_t>(p) * a.M + start + (n < count ? n : 0)) * (kSec * a.rank);
        const uint16_t* b = a.b[p] + static_cast<size_t>(adapter) * N * a.rank;
        for (int k0 = 0; k0 < kSec * a.rank; k0 += 32) {
          const int k = k0 + 8 * quarter;
          const u32x4_t none = {0, 0, 0, 0};
          u32x4_t hf = none, b0 = none, b1 = none;
          if (k < kSec * a.rank) {
            const int sec = k / a.rank, r = k - sec * a.rank;
            hf = load16(h + k);
            if (row_a < N) b0 = load16(b + static_cast<size_t>(row_a) * a.rank + r);
            if (row_a + 4 < N) b1 = load16(b + static_cast<size_t>(row_a + 4) * a.rank + r);
            if (r + 8 > rank) {  // padding, whatever it holds
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t keep = (r + 2 * e < rank ? 0xFFFFu : 0u) | (r + 2 * e + 1 < rank ? 0xFFFF0000u : 0u);
                b0[e] &= keep;
                b1[e] &= keep;
              }
            }
            b0 = section_of<T>(b0, sec);
            b1 = section_of<T>(b1, sec);
          }
          s0 = PagedBf16::mfma(b0, hf, s0);
          s1 = PagedBf16::mfma(b1, hf, s1);
        }
      }
      if (n >= count) continue;
      const uint16_t* yr = y + m * a.y_stride[p];
      uint16_t* orow = out + m * a.out_stride[p];
      if (wide && col < N) {
        const u32x4_t v = load16(yr + col);
        u32x4_t r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d0 = e < 2 ? s0[2 * e] : s1[2 * e - 4], d1 = e < 2 ? s0[2 * e + 1] : s1[2 * e - 3];
          const float y0 = T::value(static_cast<uint16_t>(v[e])), y1 = T::value(static_cast<uint16_t>(v[e] >> 16));
          r[e] = adapter < 0 ? v[e] : T::pack(__builtin_fmaf(scale, d0, y0), __builtin_fmaf(scale, d1, y1));
        }
        store16(orow + col, r);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (col + e >= N) continue;
          const uint16_t v = yr[col + e];
          orow[col + e] = adapter < 0 ? v
                                      : static_cast<uint16_t>(T::pack(
                                            __builtin_fmaf(scale, e < 4 ? s0[e] : s1[e - 4], T::value(v)), 0.0f));
        }
      }
    }
  }
}

int check_sizes(int M, int adapters) {
  if (M < 0 || adapters < 1) return CUDALM_W4A16_EINVAL;
  if (adapters > CUDALM_LORA_MAX_ADAPTERS || M > (1 << 22)) return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

size_t plan_bytes_of(int M, int adapters) {
  return sizeof(LoraPlan) + sizeof(LoraTile) * most_tiles(M, adapters) + 4 * static_cast<size_t>(M);
}

template <typename T>
int launch(const ShrinkArgs& s, const ExpandArgs& e, int tiles, hipStream_t stream) {
  constexpr int kWaves = 8;
  const long long grid = static_cast<long long>(tiles) * s.total;
  if (grid >= kMaxGemmTiles / 2) return CUDALM_W4A16_ERANGE;
  ExpandArgs x = e;
  const int steps = 1;
  long long chunks = 0;
  for (int p = 0; p < e.count; ++p) {
    x.chunk0[p] = static_cast<int>(chunks);
    chunks += (static_cast<long long>(e.N[p]) + 127) / 128;
  }
  if (chunks * tiles >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
  lora_shrink_kernel<T, 1, kWaves><<<static_cast<unsigned>(grid), 64 * kWaves, 0, stream>>>(s);
  if (const int rc = launch_status()) return rc;
  lora_expand_kernel<T, 1, 4><<<static_cast<unsigned>(chunks * tiles), 256, 0, stream>>>(x, static_cast<int>(chunks), steps);
  return launch_status();
}

}  // namespace
}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_lora_plan_bytes(int M, int adapters) {
  return check_sizes(M, adapters) == CUDALM_W4A16_OK ? plan_bytes_of(M, adapters) : 0;
}

extern "C" int cudalm_lora_plan(const int32_t* index, int M, int adapters, void* plan, size_t plan_bytes,
                                hipStream_t stream) {
  if (const int rc = check_sizes(M, adapters)) return rc;
  if (!plan || (!index && M)) return CUDALM_W4A16_ENULL;
  if (!aligned(index, 4) || !aligned(plan, 16)) return CUDALM_W4A16_EALIGN;
  if (plan_bytes < plan_bytes_of(M, adapters)) return CUDALM_W4A16_ERANGE;
  PlanArgs a = {index, static_cast<LoraPlan*>(plan), nullptr, nullptr, M, adapters};
  a.tiles = reinterpret_cast<LoraTile*>(a.plan + 1);
  a.order = reinterpret_cast<int32_t*>(a.tiles + most_tiles(M, adapters));
  const size_t lds = 4 * (static_cast<size_t>(adapters) + 1);
  lora_plan_kernel<<<1, kPlanThreads, lds, stream>>>(a);
  return launch_status();
}

extern "C" size_t cudalm_lora_workspace_bytes(int count, int M, int rank, int type) {
  if (count < 1 || count > CUDALM_LORA_MAX_PROJ || M < 0 || M > (1 << 22) || rank < 8 || rank % 8 ||
      rank > CUDALM_LORA_MAX_RANK || (type != CUDALM_LORA_BF16 && type != CUDALM_LORA_F16))
    return 0;
  return static_cast<size_t>(count) * M * rank * (type == CUDALM_LORA_BF16 ? 4 : 6);
}

extern "C" int cudalm_lora_add(const cudalm_lora_proj* projs, int count, const void* x, int64_t x_stride,
                               int K, int M, int rank, int adapters, int type, const float* scales,
                               const int32_t* ranks, const void* plan, void* workspace,
                               size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_sizes(M, adapters)) return rc;
  if (count < 1 || count > CUDALM_LORA_MAX_PROJ || K < 8 || K % 8 || rank < 8 || rank % 8 ||
      rank > CUDALM_LORA_MAX_RANK || (type != CUDALM_LORA_BF16 && type != CUDALM_LORA_F16))
    return CUDALM_W4A16_EINVAL;
  if (!projs) return CUDALM_W4A16_ENULL;
  for (int p = 0; p < count; ++p)
    if (projs[p].N < 1 || (projs[p].y == projs[p].out && projs[p].y_stride != projs[p].out_stride))
      return CUDALM_W4A16_EINVAL;
  if (M == 0) return CUDALM_W4A16_OK;
  if (!x || !plan || !workspace) return CUDALM_W4A16_ENULL;
  for (int p = 0; p < count; ++p)
    if (!projs[p].a || !projs[p].b || !projs[p].y || !projs[p].out) return CUDALM_W4A16_ENULL;
  if (!aligned(x, 16) || x_stride % 8 || !aligned(plan, 16) || !aligned(workspace, 16) ||
      !aligned(scales, 4) || !aligned(ranks, 4))
    return CUDALM_W4A16_EALIGN;
  for (int p = 0; p < count; ++p)
    if (!aligned(projs[p].a, 16) || !aligned(projs[p].b, 16) || !aligned(projs[p].y, 2) ||
        !aligned(projs[p].out, 2))
      return CUDALM_W4A16_EALIGN;
  if (workspace_bytes < cudalm_lora_workspace_bytes(count, M, rank, type)) return CUDALM_W4A16_ERANGE;
  const int tiles = most_tiles(M, adapters);
  ShrinkArgs s = {};
  s.plan = static_cast<const LoraPlan*>(plan);
  s.tiles = reinterpret_cast<const LoraTile*>(s.plan + 1);
  s.order = reinterpret_cast<const int32_t*>(s.tiles + tiles);
  s.ranks = ranks;
  s.x = static_cast<const uint16_t*>(x);
  s.h = static_cast<uint16_t*>(workspace);
  s.x_stride = x_stride;
  s.K = K;
  s.M = M;
  s.rank = rank;
  s.rank_tiles = (rank + 15) / 16;
  s.total = s.rank_tiles * count;
  ExpandArgs e = {};
  e.plan = s.plan;
  e.tiles = s.tiles;
  e.order = s.order;
  e.ranks = ranks;
  e.scales = scales;
  e.h = s.h;
  e.count = count;
  e.M = M;
  e.rank = rank;
  for (int p = 0; p < count; ++p) {
    s.a[p] = static_cast<const uint16_t*>(projs[p].a);
    e.b[p] = static_cast<const uint16_t*>(projs[p].b);
    e.y[p] = static_cast<const uint16_t*>(projs[p].y);
    e.out[p] = static_cast<uint16_t*>(projs[p].out);
    e.y_stride[p] = projs[p].y_stride;
    e.out_stride[p] = projs[p].out_stride;
    e.N[p] = projs[p].N;
    if (aligned(projs[p].y, 16) && aligned(projs[p].out, 16) && projs[p].y_stride % 8 == 0 &&
        projs[p].out_stride % 8 == 0 && projs[p].N % 8 == 0)
      e.wide |= 1 << p;
  }
  return type == CUDALM_LORA_BF16 ? launch<PagedBf16>(s, e, tiles, stream) : launch<PagedF16>(s, e, tiles, stream);
}
