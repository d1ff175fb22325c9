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

#include "paged_decode_body.h"

namespace cudalm_hip {
namespace {

// WV waves: RT tiles of rows, WV / RT slices.
template <typename T, int D, int RT, int WV, bool RANGES>
__global__ __launch_bounds__(64 * WV, 2) void paged_decode_kernel(const DecodeArgs a) {
  __shared__ DecodeLds<D, RT, WV> lds;
  paged_decode_body<T, D, RT, WV, RANGES>(a, lds, blockIdx.x);
}

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
