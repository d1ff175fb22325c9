// Low-rank adapters of many requests beside shared projections: two products with a
// rank between them, h = A x and y + s B h, over tiles of up to 16 rows that have the
// same adapter.
//
// Rows are the columns of the matrix products (16x16x32), so that an adapter's factors
// are read as they lie, 16 bytes of a row per lane, and one tile reads them once for
// its rows. h is summed in fp32 over the waves of a workgroup. The second product takes
// bf16 operands only: h = hh + hl, two bf16 numbers, keep 16 of its bits and all of fp32's
// range, which fp16 would not; fp16 factors are split in the same way, b = bh + bl, exactly.
// h is therefore held as sections of `rank` numbers each along the summed index,
//
//   h:  hh | hl            (fp16: hh | hl | hh without Inf and NaN)
//   b:  b  | b without Inf and NaN          (fp16: bh | bh without .. | bl)
//
// so that the products of a section meet and Inf times 0 comes up only where the
// unsplit factors have it.

#include "cudalm_lora.h"

#include "paged_device.h"
#include "row_places.h"

namespace cudalm_hip {
namespace {

constexpr int kRows = 16;   // of a tile
constexpr int kWaves = 8;   // of a workgroup
constexpr int kPlanThreads = 1024;

// A plan: the number of tiles, three words, the tiles, the 16 rows of each.
struct LoraTile {
  int adapter, count;  // adapter -1: rows of none
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
  int32_t* rows;
  int M, adapters;
};

// For every lane with a number a (a < 0: none): how much counter[a] was before the lanes
// up to this one added one each. Lanes of one number, as prompts have them, add in one; others each for
// themselves (64 rows of 48 adapters: 3.0 us, 7.1 with an addition of all of a number's lanes in turn).
__device__ __forceinline__ int claim(int* counter, int a) {
  const int lane = threadIdx.x & 63;
  const uint64_t real = __ballot(a >= 0);
  if (real == 0) return 0;
  const int leader = __builtin_ctzll(real), one = __builtin_amdgcn_readlane(a, leader);
  if (__ballot(a == one) != real) return a >= 0 ? atomicAdd(&counter[a], 1) : 0;
  int base = 0;
  if (lane == leader) base = atomicAdd(&counter[one], static_cast<int>(__popcll(real)));
  base = __builtin_amdgcn_readlane(base, leader);
  return base + static_cast<int>(__popcll(real & ((1ULL << lane) - 1)));
}

// One workgroup: rows per adapter, the tiles of each, and their rows. Which of two rows of an
// adapter comes first is open; no result depends on it, since every row is a column of its own
// in the products. Latency: 3 us for one row or 64 rows of 48 adapters, 9 for 4001 rows; a
// step has one for all of its layers.
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const PlanArgs a) {
  extern __shared__ int counter[];  // [adapters + 1], the last for rows of none; and the first tiles
  __shared__ int tiles_of[kPlanThreads / 64];
  const int groups = a.adapters + 1, lane = threadIdx.x & 63, wave = wave_id();
  int* first_tile = counter + groups;
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
  int tiles = 0;
  for (int i = from; i < to; ++i) tiles += (counter[i] + kRows - 1) / kRows;
  int before = tiles;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const int t = __shfl_up(before, x);
    if (lane >= x) before += t;
  }
  if (lane == 63) tiles_of[wave] = before;
  __syncthreads();
  before -= tiles;
  for (int w = 0; w < wave; ++w) before += tiles_of[w];
  if (threadIdx.x == kPlanThreads - 1) a.plan->tiles = before + tiles;
  for (int i = from; i < to; ++i) {
    const int n = counter[i];
    counter[i] = 0;
    first_tile[i] = before;
    for (int r = 0; r < n; r += kRows)
      a.tiles[before++] = {i < a.adapters ? i : -1, n - r < kRows ? n - r : kRows};
  }
  __syncthreads();
  for (int m0 = 64 * wave; m0 < a.M; m0 += kPlanThreads) {
    const int m = m0 + lane, group = m < a.M ? group_of(m) : -1;
    const int at = claim(counter, group);
    if (group >= 0) a.rows[first_tile[group] * kRows + at] = m;
  }
}

struct LoraArgs {
  const LoraPlan* plan;
  const LoraTile* tiles;
  const int32_t* rows;
  const int32_t* ranks;  // or NULL
  const float* scales;   // or NULL
  const uint16_t* x;
  const uint16_t* a[CUDALM_LORA_MAX_PROJ];
  const uint16_t* b[CUDALM_LORA_MAX_PROJ];
  const uint16_t* y[CUDALM_LORA_MAX_PROJ];
  uint16_t* out[CUDALM_LORA_MAX_PROJ];
  long long x_stride, y_stride[CUDALM_LORA_MAX_PROJ], out_stride[CUDALM_LORA_MAX_PROJ];
  int N[CUDALM_LORA_MAX_PROJ], chunk0[CUDALM_LORA_MAX_PROJ];  // first chunk of columns of each
  int count, K, rank, wide;  // wide: a bit for each projection whose rows go 16 bytes at a time
  int chunks, steps, most_tiles;  // chunks of all; a chunk is `steps` x kColumns
};

template <typename T>
constexpr int kSections = T::kExp == PagedBf16::kExp ? 2 : 3;

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < __builtin_inff() ? x : 0.0f; }

// A number as bf16 and the rest of it, which is 0 beside Inf and NaN.
__device__ __forceinline__ void split(float x, float& hi, float& lo) {
  hi = bf16_lo(f32_to_bf16_rne(x));
  lo = finite_or_zero(x - hi);
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

// A tile of rows and a chunk of a projection's columns: h of the tile, its waves splitting K,
// then the columns. Every chunk of a tile makes h anew: its factors and the rows' activations
// come from the L2 of the tile's XCD then, where a launch of its own for h would cost what these
// calls take. Lane (n, quarter) of a wave holds columns 8 quarter .. + 7 of row n, from two
// products whose rows stand for columns 8 (i / 4) + 4 f + i % 4; and 32 further. RT: rank tiles of 16 at a
// time; up to 16 RT ranks, or any number where RT is 4.
// Steps are bound by a chain of latencies: rows and tile 2 us, A and x 2, h 1, columns 1 to 2. One row of
// K = 1024 on q, k, v of 5120 columns in all, rank 16: 5.0 us; 64 rows of 48 adapters 6.8 (two launches
// 8.5); 33 rows, gate and up of 3584, rank 64, fp16: 10.3. 4001 rows of 5 adapters, K = 3584, N = 1024, rank
// 32: 15 us, 3 TB/s, of which x times A takes 8.6: four rounds of loads, a workgroup's waves two pieces
// of 64 each, in turn with their products (a round ahead: 15.2, and spills; sixteen waves: 18).
template <typename T, int RT, int HALVES>
__global__ __launch_bounds__(64 * kWaves, RT < 4 ? 4 : 2) void lora_kernel(const LoraArgs a) {
  constexpr int kColumns = 32 * HALVES * kWaves, kF = 2 * HALVES;
  constexpr int kSec = kSections<T>, kMost = RT < 4 ? 16 * RT : CUDALM_LORA_MAX_RANK;
  // a wave's lines of x and A on their way to the operands, then its sums, then results on
  // their way to lines
  __shared__ union {
    u32x4_t lines[kWaves][1 + RT][128];
    float sums[kWaves][RT][256];
    f32x4_t columns[kWaves][HALVES * 128];
  } shared;
  alignas(16) __shared__ uint16_t hidden[kRows * (kSec * kMost + 8)];  // rows of 8 more than they need: other banks
  // the chunks of a tile in one XCD, one after the other
  const int t = blockIdx.x / 8 / a.chunks * 8 + blockIdx.x % 8, chunk = blockIdx.x / 8 % a.chunks;
  const int lane = threadIdx.x & 63, wave = wave_id(), n = lane & 15, quarter = lane >> 4;
  // rows whose lines this lane loads: of x by eight lanes, of y by 4 HALVES
  constexpr int kLanes = 4 * HALVES;
  const int of_eight = lane >> 3, of_lanes = lane / kLanes;
  int line_row[2] = {0, 0}, out_row[HALVES] = {};
  if (t < a.most_tiles) {
    line_row[0] = a.rows[t * kRows + of_eight];
    line_row[1] = a.rows[t * kRows + 8 + of_eight];
    if (HALVES == 1) out_row[0] = a.rows[t * kRows + of_lanes];
  }
  if (t >= load_uniform(&a.plan->tiles)) return;
  const int adapter = load_uniform(&a.tiles[t].adapter), count = load_uniform(&a.tiles[t].count);
  int p = 0;
  while (p + 1 < a.count && chunk >= a.chunk0[p + 1]) ++p;
  const uint16_t* y = a.y[p];
  uint16_t* out = a.out[p];
  if (adapter < 0 && y == out) return;
  const int N = a.N[p], R = a.rank, pitch = kSec * R + 8;
  const bool wide = (a.wide >> p) & 1;
  const u32x4_t none = {0, 0, 0, 0};
  int rank = 0;
  if (adapter >= 0) rank = a.ranks ? load_uniform(a.ranks + adapter) : R;
  rank = rank < 0 ? 0 : rank < R ? rank : R;
  const int first_row = __builtin_amdgcn_readfirstlane(line_row[0]);
  if (of_eight >= count) line_row[0] = first_row;  // a copy of it
  if (8 + of_eight >= count) line_row[1] = first_row;
  const int out_col = 8 * (lane % kLanes);
  const uint16_t* yr[HALVES];
  uint16_t* orow[HALVES];
  bool there[HALVES];
#pragma unroll
  for (int j = 0; j < HALVES; ++j) {
    there[j] = 8 * j + of_lanes < count;
    const int m = HALVES == 2 ? line_row[j] : there[j] ? out_row[j] : first_row;
    yr[j] = y + m * a.y_stride[p] + out_col;
    orow[j] = out + m * a.out_stride[p] + out_col;
  }

  // The columns' operands: pieces of 32 along the summed index, which is a section at a time (whole
  // ranks of 32: a load serves all of them) or all sections in a row. One is loaded ahead, the
  // first before h is made.
  const bool whole = R % 32 == 0;
  const int pieces = adapter < 0 ? 1 : whole ? R / 32 : (kSec * R + 31) / 32;
  const uint16_t* factor_b = a.b[p] + static_cast<size_t>(adapter < 0 ? 0 : adapter) * N * R;
  const int first = (chunk - a.chunk0[p]) * a.steps * kColumns + 32 * HALVES * wave;
  int next_step = 0, next_piece = 0;
  u32x4_t factor[kF] = {}, old[HALVES] = {};
  auto load_next = [&]() {
    const int n0 = first + next_step * kColumns;
    if (next_step >= a.steps || n0 >= N) return;
    const int k = 32 * next_piece + 8 * quarter, r = whole ? k : k % R, row = n0 + 8 * (n >> 2) + (n & 3);
    const bool in = adapter >= 0 && k < (whole ? R : kSec * R) && r < rank;
#pragma unroll
    for (int f = 0; f < kF; ++f) {  // columns 4 (f % 2) of eight further, of the half f / 2
      const int at = row + 4 * (f % 2) + 32 * (f / 2);
      factor[f] = in && at < N ? load16(factor_b + static_cast<size_t>(at) * R + r) : none;
    }
    if (in && r + 8 > rank) {  // padding, whatever it holds
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t keep = (r + 2 * e < rank ? 0xFFFFu : 0u) | (r + 2 * e + 1 < rank ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int f = 0; f < kF; ++f) factor[f][e] &= keep;
      }
    }
    if (wide && next_piece == 0 && n0 + out_col < N)
#pragma unroll
      for (int j = 0; j < HALVES; ++j)
        if (there[j]) old[j] = load16(yr[j] + n0);
    if (++next_piece == pieces) next_piece = 0, ++next_step;
  };
  load_next();

  if (adapter >= 0) {
    // 64 numbers of 16 rows at a time, a line of each: eight lanes load one (lanes of an operand
    // that read 16 bytes of 16 rows each take a cycle of the cache apiece: 4001 rows, K = 3584,
    // rank 32 took 18 us, 15 so), LDS turns them into operands. Chunk c of row r lies at
    // c ^ r / 2 there, or rows would meet in the same banks.
    const uint16_t* x[2];
    int at[2];  // of this lane's chunk in its lines
    const uint16_t* factor_a = a.a[p] + static_cast<size_t>(adapter) * R * a.K;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      at[j] = 8 * ((lane & 7) ^ (4 * j + (of_eight >> 1)));
      x[j] = a.x + line_row[j] * a.x_stride + at[j];
    }
    u32x4_t(*lines)[128] = shared.lines[wave];
    for (int r0 = 0; r0 < R; r0 += 16 * RT) {
      f32x4_t sum[RT];
      const uint16_t* row_a[RT][2];
      bool real[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        sum[i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = r0 + 16 * i + 8 * j + of_eight;
          real[i][j] = r < rank;
          row_a[i][j] = factor_a + static_cast<size_t>(real[i][j] ? r : 0) * a.K + at[j];
        }
      }
      for (int k0 = 64 * wave; k0 < a.K; k0 += 2 * 64 * kWaves) {
        u32x4_t xf[2][2], af[2][RT][2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int k = k0 + s * 64 * kWaves;
            const bool in = k + at[j] < a.K;
            xf[s][j] = in ? load16(x[j] + k) : none;
#pragma unroll
            for (int i = 0; i < RT; ++i) af[s][i][j] = in && real[i][j] ? load16(row_a[i][j] + k) : none;
          }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            lines[0][64 * j + lane] = xf[s][j];
#pragma unroll
            for (int i = 0; i < RT; ++i) lines[1 + i][64 * j + lane] = af[s][i][j];
          }
          wave_lds_sync();
#pragma unroll
          for (int c = 0; c < 8; c += 4) {
            const int place = 8 * n + ((c + quarter) ^ (n >> 1));
            const u32x4_t b = lines[0][place];
#pragma unroll
            for (int i = 0; i < RT; ++i) sum[i] = T::mfma(lines[1 + i][place], b, sum[i]);
          }
          wave_lds_sync();
        }
      }
      __syncthreads();  // lines have been read
#pragma unroll
      for (int i = 0; i < RT; ++i)  // rank 4 quarter + e of row n
        *reinterpret_cast<f32x4_t*>(&shared.sums[wave][i][16 * n + 4 * quarter]) = sum[i];
      __syncthreads();
      for (int i = threadIdx.x; i < RT * 256; i += 64 * kWaves) {
        const int r = r0 + i / 256 * 16 + i % 16, row = i / 16 % 16;
        if (r >= R) continue;
        float v = 0, hi, lo;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += shared.sums[w][i / 256][i % 256];
        if (r >= rank) v = 0;  // padding: its zeros times Inf of x are NaN
        split(v, hi, lo);
        uint16_t* h = hidden + row * pitch + r;
        h[0] = static_cast<uint16_t>(f32_to_bf16_rne(hi));
        h[R] = static_cast<uint16_t>(f32_to_bf16_rne(lo));
        if (kSec == 3) h[2 * R] = static_cast<uint16_t>(f32_to_bf16_rne(finite_or_zero(hi)));
      }
      __syncthreads();  // sums have been read, h is there
    }
  }

  const float scale = adapter >= 0 && a.scales ? a.scales[adapter] : 1.0f;
  const uint16_t* hrow = hidden + n * pitch;
#pragma unroll 1
  for (int step = 0; step < a.steps; ++step) {
    const int n0 = first + step * kColumns;
    if (n0 >= N) break;
    u32x4_t before[HALVES];
#pragma unroll
    for (int half = 0; half < HALVES; ++half) before[half] = old[half];
    f32x4_t sum[kF];
#pragma unroll
    for (int f = 0; f < kF; ++f) sum[f] = f32x4_t{0, 0, 0, 0};
#pragma unroll 1
    for (int piece = 0; piece < pieces; ++piece) {
      u32x4_t b[kF];
#pragma unroll
      for (int f = 0; f < kF; ++f) b[f] = factor[f];
      const int k = 32 * piece + 8 * quarter;
      load_next();
      if (adapter < 0) break;
      if (whole) {
#pragma unroll
        for (int sec = 0; sec < kSec; ++sec) {
          const u32x4_t hf = load16(hrow + sec * R + k);
#pragma unroll
          for (int f = 0; f < kF; ++f) sum[f] = PagedBf16::mfma(section_of<T>(b[f], sec), hf, sum[f]);
        }
      } else {
        const int sec = k / R;
        const u32x4_t hf = sec < kSec ? load16(hrow + k) : none;
#pragma unroll
        for (int f = 0; f < kF; ++f) sum[f] = PagedBf16::mfma(section_of<T>(b[f], sec), hf, sum[f]);
      }
    }
    // to rows of 32 HALVES columns, four of them at a place exchanged by the row
    f32x4_t* columns = shared.columns[wave];
    if (adapter >= 0) {
#pragma unroll
      for (int f = 0; f < kF; ++f) {
        const int c = 8 * (f / 2) + 2 * quarter + f % 2;
        columns[8 * HALVES * n + (c ^ (n & (8 * HALVES - 1)))] = sum[f];
      }
      wave_lds_sync();
    }
#pragma unroll
    for (int j = 0; j < HALVES; ++j) {
      const int row = 8 * j + of_lanes, c = out_col / 4, col = n0 + out_col;
      const f32x4_t d0 = columns[8 * HALVES * row + (c ^ (row & (8 * HALVES - 1)))];
      const f32x4_t d1 = columns[8 * HALVES * row + ((c + 1) ^ (row & (8 * HALVES - 1)))];
      if (!there[j] || col >= N) continue;
      if (wide) {
        u32x4_t r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t v = before[j][e];
          const float y0 = T::value(static_cast<uint16_t>(v)), y1 = T::value(static_cast<uint16_t>(v >> 16));
          const float x0 = e < 2 ? d0[2 * e] : d1[2 * e - 4], x1 = e < 2 ? d0[2 * e + 1] : d1[2 * e - 3];
          r[e] = rank == 0 ? v : T::pack(__builtin_fmaf(scale, x0, y0), __builtin_fmaf(scale, x1, y1));
        }
        store16(orow[j] + n0, r);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (col + e >= N) continue;
          const uint16_t w = yr[j][n0 + e];
          const float d = e < 4 ? d0[e] : d1[e - 4];
          orow[j][n0 + e] = rank == 0 ? w : static_cast<uint16_t>(T::pack(__builtin_fmaf(scale, d, T::value(w)), 0.0f));
        }
      }
    }
    wave_lds_sync();
  }
}

int check_sizes(int M, int adapters) {
  if (M < 0 || adapters < 1) return CUDALM_W4A16_EINVAL;
  if (adapters > CUDALM_LORA_MAX_ADAPTERS || M > (1 << 22)) return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

size_t plan_bytes_of(int M, int adapters) {
  return sizeof(LoraPlan) + (sizeof(LoraTile) + 4 * kRows) * static_cast<size_t>(most_tiles(M, adapters));
}

template <typename T, int RT>
int launch(LoraArgs& a, int tiles, hipStream_t stream) {
  const long long groups = (static_cast<long long>(tiles) + 7) / 8 * 8;
  // Columns per workgroup: 32 for every wave, then 64, then steps of them, until there are
  // no more than three workgroups for a CU, or two where h costs each of them more than 128 KB
  // (64 rows of 48 adapters, rank 16, K = 1024: 7.0 us with three, 8.3 with two; 4001 rows,
  // rank 32, K = 3584: 528 workgroups, which three allow, 20; 264 of two steps, which is the next
  // number below two's limit and one for a CU, 15). `tiles` is the most that a plan can have:
  // adapters that no row has count in it and leave those in use fewer workgroups (1024 rows of one
  // adapter, K = N = 4096, rank 16: 12.6 us among 8 adapters, 13.4 among 64, 20.2 among 512).
  const int limit = (static_cast<long long>(a.K) * (kRows + a.rank) > 65536 ? 2 : 3) * cu_count();
  long long chunks;
  int halves = 1;
  for (a.steps = 1;; a.steps += 1 + a.steps / 8) {
    const long long span = 32LL * halves * kWaves * a.steps;
    chunks = 0;
    for (int p = 0; p < a.count; ++p) {
      a.chunk0[p] = chunks < kMaxGemmTiles ? static_cast<int>(chunks) : 0;
      chunks += (a.N[p] + span - 1) / span;
    }
    if (chunks == a.count || groups * chunks <= limit) break;
    if (halves == 1) halves = 2, a.steps = 0;
  }
  if (groups * chunks >= kMaxGemmTiles / 4) return CUDALM_W4A16_ERANGE;
  a.chunks = static_cast<int>(chunks);
  a.most_tiles = tiles;
  auto kernel = halves == 1 ? lora_kernel<T, RT, 1> : lora_kernel<T, RT, 2>;
  kernel<<<static_cast<unsigned>(groups * chunks), 64 * kWaves, 0, stream>>>(a);
  return launch_status();
}

template <typename T>
int launch_rank(LoraArgs& a, int tiles, hipStream_t stream) {
  return a.rank <= 16 ? launch<T, 1>(a, tiles, stream)
         : a.rank <= 32 ? launch<T, 2>(a, tiles, stream)
                        : launch<T, 4>(a, tiles, stream);
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
  a.rows = reinterpret_cast<int32_t*>(a.tiles + most_tiles(M, adapters));
  const size_t lds = 8 * (static_cast<size_t>(adapters) + 1);
  lora_plan_kernel<<<1, kPlanThreads, lds, stream>>>(a);
  return launch_status();
}

extern "C" int cudalm_lora_add(const cudalm_lora_proj* projs, int count, const void* x, int64_t x_stride,
                               int K, int M, int rank, int adapters, int type, const float* scales,
                               const int32_t* ranks, const void* plan, hipStream_t stream) {
  if (const int rc = check_sizes(M, adapters)) return rc;
  if (count < 1 || count > CUDALM_LORA_MAX_PROJ || K < 8 || K % 8 || rank < 8 || rank % 8 ||
      rank > CUDALM_LORA_MAX_RANK || (type != CUDALM_LORA_BF16 && type != CUDALM_LORA_F16))
    return CUDALM_W4A16_EINVAL;
  if (!projs) return CUDALM_W4A16_ENULL;
  for (int p = 0; p < count; ++p) {
    if (projs[p].N < 1 || (projs[p].y == projs[p].out && projs[p].y_stride != projs[p].out_stride))
      return CUDALM_W4A16_EINVAL;
    // workgroups read x and y while others write: a result's place is its own
    const int64_t step = projs[p].out_stride < 0 ? -projs[p].out_stride : projs[p].out_stride;
    if (M > 1 && step < projs[p].N) return CUDALM_W4A16_EINVAL;
    if (projs[p].out && projs[p].out == x) return CUDALM_W4A16_EINVAL;
    for (int o = 0; o < count && projs[p].out; ++o)
      if (o != p && (projs[p].out == projs[o].out || projs[p].out == projs[o].y)) return CUDALM_W4A16_EINVAL;
  }
  for (int p = 0; p < count; ++p)
    if (projs[p].N > (1 << 28)) return CUDALM_W4A16_ERANGE;
  if (M == 0) return CUDALM_W4A16_OK;
  if (!x || !plan) return CUDALM_W4A16_ENULL;
  for (int p = 0; p < count; ++p)
    if (!projs[p].a || !projs[p].b || !projs[p].y || !projs[p].out) return CUDALM_W4A16_ENULL;
  if (!aligned(x, 16) || x_stride % 8 || !aligned(plan, 16) || !aligned(scales, 4) || !aligned(ranks, 4))
    return CUDALM_W4A16_EALIGN;
  LoraArgs a = {};
  const int tiles = most_tiles(M, adapters);
  a.plan = static_cast<const LoraPlan*>(plan);
  a.tiles = reinterpret_cast<const LoraTile*>(a.plan + 1);
  a.rows = reinterpret_cast<const int32_t*>(a.tiles + tiles);
  a.ranks = ranks;
  a.scales = scales;
  a.x = static_cast<const uint16_t*>(x);
  a.x_stride = x_stride;
  a.count = count;
  a.K = K;
  a.rank = rank;
  for (int p = 0; p < count; ++p) {
    const cudalm_lora_proj& q = projs[p];
    if (!aligned(q.a, 16) || !aligned(q.b, 16) || !aligned(q.y, 2) || !aligned(q.out, 2)) return CUDALM_W4A16_EALIGN;
    a.a[p] = static_cast<const uint16_t*>(q.a);
    a.b[p] = static_cast<const uint16_t*>(q.b);
    a.y[p] = static_cast<const uint16_t*>(q.y);
    a.out[p] = static_cast<uint16_t*>(q.out);
    a.y_stride[p] = q.y_stride;
    a.out_stride[p] = q.out_stride;
    a.N[p] = q.N;
    if (aligned(q.y, 16) && aligned(q.out, 16) && q.y_stride % 8 == 0 && q.out_stride % 8 == 0 && q.N % 8 == 0)
      a.wide |= 1 << p;
  }
  // nor does a result lie over a part of what is read, or of another one
  for (int p = 0; p < count; ++p) {
    const RowGrid out = {projs[p].out, M, projs[p].out_stride, 1, 0, projs[p].N};
    if (places_meet(out, {x, M, x_stride, 1, 0, K})) return CUDALM_W4A16_EINVAL;
    for (int o = 0; o < count; ++o) {
      const cudalm_lora_proj& q = projs[o];
      if ((o != p || q.y != q.out) && places_meet(out, {q.y, M, q.y_stride, 1, 0, q.N})) return CUDALM_W4A16_EINVAL;
      if (o > p && places_meet(out, {q.out, M, q.out_stride, 1, 0, q.N})) return CUDALM_W4A16_EINVAL;
    }
  }
  return type == CUDALM_LORA_BF16 ? launch_rank<PagedBf16>(a, tiles, stream) : launch_rank<PagedF16>(a, tiles, stream);
}
