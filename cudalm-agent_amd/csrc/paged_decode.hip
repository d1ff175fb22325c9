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
// A workgroup of four waves takes RT tiles of 16 rows and 4 / RT slices of the
// tokens of its split; slices are joined in LDS, splits by a second kernel.

#include <cstdint>

#include "paged_device.h"

namespace cudalm_hip {
namespace {

constexpr int kTile = 32;      // tokens per step of a wave
constexpr int kTileShift = 5;

struct DecodeArgs {
  PagedView kv;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  void* out;
  float* part_o;    // [bh][splits][rows][D], NULL: one split, straight to out
  float* part_ml;   // [bh][splits][rows][2]
  float* final_ml;  // [bh][rows][2] or NULL
  float* scores;    // [bh][rows][score_pitch] (times scale log2 e) or NULL
  long long token_stride, head_stride;
  float scale_log2;
  int new_tokens, group, rows, splits, least, window, sinks, score_pitch;
};

template <typename T, int D, int RT>
__global__ __launch_bounds__(256, 2) void paged_decode_kernel(const DecodeArgs a) {
  constexpr int KK = D / 32, DT = D / 16, SL = 4 / RT;
  constexpr int kPitch = D + 4;
  __shared__ float obuf[2][16 * kPitch];
  __shared__ float mlbuf[4][2][16];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int n = lane & 15, quarter = lane >> 4;
  const int rt = wave % RT, slice = wave / RT;

  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int bh = id % (a.kv.batch * a.kv.kv_heads), zr = id / (a.kv.batch * a.kv.kv_heads);
  const int b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;

  const int length = a.kv.uniform_length(b), first = length - a.new_tokens;
  const PagedTiles tiles(length, first, length - 1, a.window, a.sinks, kTileShift);
  const int per = tiles_per_split(tiles.count, a.splits, a.least, SL);
  const int begin = split * per, end = begin + per < tiles.count ? begin + per : tiles.count;
  if (a.part_o && begin >= end) return;  // the join knows how many splits there are

  // this lane's row
  const int row = (zr * RT + rt) * 16 + n;
  const bool real = row < a.rows;
  const int j = row / a.group;
  const int pos = real ? first + j : -1;

  u32x4_t qf[KK];
  {
    const uint16_t* qp = a.q +
                         (static_cast<long long>(b) * a.new_tokens + (real ? j : 0)) * a.token_stride +
                         (static_cast<long long>(h) * a.group + (real ? row - j * a.group : 0)) *
                             a.head_stride +
                         8 * quarter;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = *reinterpret_cast<const u32x4_t*>(qp + 32 * kk);
      if (!real) qf[kk] = u32x4_t{0, 0, 0, 0};
    }
  }

  f32x4_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_t{0, 0, 0, 0};
  float m = kLowest, l = 0;

  const int P = 1 << a.kv.page_shift;
  const size_t page_elems = (static_cast<size_t>(P) * D) * a.kv.kv_heads;
  const size_t head_elems = static_cast<size_t>(P) * D * h;
  const int ktok = 8 * (n >> 2) + (n & 3);  // token of K row n in half 0
  u32x4_t kf[2][KK], vf[DT];

  // The pages of a tile's two halves, and whether every row sees all of it.
  int t0 = 0, pa = -1, pb = -1;
  auto look_up = [&](int i) {
    t0 = tiles.tile(i) << kTileShift;
    pa = a.kv.uniform_page(b, t0 >> a.kv.page_shift);
    pb = a.kv.uniform_page(b, (t0 + 16) >> a.kv.page_shift);
    return pa >= 0 && pb >= 0 && t0 + kTile - 1 <= first &&
           (a.window <= 0 || t0 > length - 1 - a.window || t0 + kTile - 1 < a.sinks);
  };
  auto load_k = [&]() {
    const int pg = n < 8 ? pa : pb;
    const uint16_t* kp = a.k + (pg < 0 ? 0 : pg) * page_elems + head_elems +
                         static_cast<size_t>((t0 + ktok) & (P - 1)) * D + 8 * quarter;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int f = 0; f < 2; ++f)
        kf[f][kk] = *reinterpret_cast<const u32x4_t*>(kp + 4 * f * D + 32 * kk);
  };
  auto load_v = [&]() {
    const int pg = quarter < 2 ? pa : pb;
    const uint16_t* vp = a.v + (pg < 0 ? 0 : pg) * page_elems + head_elems +
                         static_cast<size_t>((t0 + 8 * quarter) & (P - 1)) * D + 8 * n;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vf[dt] = *reinterpret_cast<const u32x4_t*>(vp + 128 * dt);
  };
  float t[8];  // this lane's scores: its row, tokens 8 quarter .. 8 quarter + 7
  auto scores = [&]() {
    f32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      s0 = T::mfma(kf[0][kk], qf[kk], s0);
      s1 = T::mfma(kf[1][kk], qf[kk], s1);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = s0[e] * a.scale_log2;
      t[4 + e] = s1[e] * a.scale_log2;
    }
  };
  auto keep_scores = [&](int tile0) {
    if (!a.scores || !real || tile0 + kTile > a.score_pitch) return;
    float* sp = a.scores + (static_cast<size_t>(bh) * a.rows + row) * a.score_pitch + tile0 +
                8 * quarter;
    *reinterpret_cast<f32x4_t*>(sp) = f32x4_t{t[0], t[1], t[2], t[3]};
    *reinterpret_cast<f32x4_t*>(sp + 4) = f32x4_t{t[4], t[5], t[6], t[7]};
  };
  u32x4_t pf;
  auto softmax = [&]() {
    float top = t[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, t[e]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
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

  // Tiles that are seen whole: the next one's keys load while this one's
  // weights are made, its values while the scores are.
  int i = begin + slice;
  while (i < end && !look_up(i)) i += SL;
  if (i < end) load_k();
  while (i < end) {
    load_v();
    const int tile0 = t0;
    scores();
    do i += SL;
    while (i < end && !look_up(i));
    if (i < end) load_k();
    keep_scores(tile0);
    softmax();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma(vf[dt], pf, o[dt]);
  }
  // The others: at the ends of the sequence, the window and the sinks, and
  // where pages are absent.
#pragma unroll 1
  for (i = begin + slice; i < end; i += SL) {
    if (look_up(i)) continue;
    load_k();
    scores();
    const bool has = (quarter < 2 ? pa : pb) >= 0;
    uint32_t seen = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool sees = has && paged_sees(t0 + 8 * quarter + e, pos, a.window, a.sinks);
      seen |= sees ? 1u << e : 0u;
      t[e] = sees ? t[e] : -__builtin_inff();
    }
    keep_scores(t0);
    softmax();
    load_v();
    // values of tokens that no row here sees may be anything: take them out
    uint32_t some = seen, bad = 0;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) some |= __shfl_xor(static_cast<int>(some), x);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        vf[dt][w] &= ((some >> (2 * w)) & 1 ? 0xFFFFu : 0u) |
                     ((some >> (2 * w + 1)) & 1 ? 0xFFFF0000u : 0u);
      bad |= special_bits<T>(vf[dt]);
    }
    if (__any(bad != 0)) {
      const u32x4_t sees = seen_operand<T>(seen);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4_t up = T::mfma(special_part<T>(vf[dt], ~0u), sees, f32x4_t{0, 0, 0, 0});
        const f32x4_t down = T::mfma(special_part<T>(vf[dt], 0), sees, f32x4_t{0, 0, 0, 0});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[dt][e] += (up[e] > 0 ? __builtin_inff() : 0.0f) + (down[e] > 0 ? -__builtin_inff() : 0.0f);
        vf[dt] = finite_part<T>(vf[dt]);
        __builtin_amdgcn_sched_barrier(0);  // few registers over speed here
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma(vf[dt], pf, o[dt]);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // join the slices: the upper half of the waves hands its sums down
  if (SL > 1) {
    if (quarter == 0) mlbuf[wave][0][n] = m, mlbuf[wave][1][n] = l;
    __syncthreads();
    float all = m;
#pragma unroll
    for (int s = 0; s < SL; ++s) all = fmaxf(all, mlbuf[s * RT + rt][0][n]);
    l = 0;
#pragma unroll
    for (int s = 0; s < SL; ++s)
      l += mlbuf[s * RT + rt][1][n] * exp2_fast(mlbuf[s * RT + rt][0][n] - all);
    const float r = exp2_fast(m - all);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= r;
    m = all;
#pragma unroll
    for (int half = SL / 2; half > 0; half >>= 1) {
      if (slice >= half && slice < 2 * half) {
        float* p = obuf[(slice - half) * RT + rt] + n * kPitch + 4 * quarter;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(p + 16 * dt) = o[dt];
      }
      __syncthreads();
      if (slice < half) {
        const float* p = obuf[slice * RT + rt] + n * kPitch + 4 * quarter;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] += *reinterpret_cast<const f32x4_t*>(p + 16 * dt);
      }
      __syncthreads();
    }
    if (slice > 0) return;
  }
  if (!real) return;
  if (a.part_o) {
    const size_t at = (static_cast<size_t>(bh) * a.splits + split) * a.rows + row;
    float* p = a.part_o + at * D + 4 * quarter;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(p + 16 * dt) = o[dt];
    if (quarter == 0) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
    return;
  }
  if (a.final_ml && quarter == 0) {
    const size_t at = static_cast<size_t>(bh) * a.rows + row;
    a.final_ml[2 * at] = m;
    a.final_ml[2 * at + 1] = l;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int heads = a.group * a.kv.kv_heads;
  uint16_t* y = static_cast<uint16_t*>(a.out) +
                ((static_cast<size_t>(b) * a.new_tokens + j) * heads + h * a.group + row - j * a.group) *
                    D +
                4 * quarter;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    *reinterpret_cast<u32x2_t*>(y + 16 * dt) =
        u32x2_t{T::pack(o[dt][0] * inv, o[dt][1] * inv), T::pack(o[dt][2] * inv, o[dt][3] * inv)};
}

// One workgroup per row: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over
// the splits of the row's sequence, a quarter of them per wave.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const DecodeArgs a, int unit) {
  constexpr int E = D / 64;
  __shared__ float obuf[4][D];
  __shared__ float lbuf[4];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int bh = blockIdx.x / a.rows, row = blockIdx.x % a.rows;
  const int b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;
  const int length = a.kv.uniform_length(b), first = length - a.new_tokens;
  const PagedTiles tiles(length, first, length - 1, a.window, a.sinks, kTileShift);
  const int per = tiles_per_split(tiles.count, a.splits, a.least, unit);
  const int count = (tiles.count + per - 1) / per;
  const size_t at = static_cast<size_t>(bh) * a.splits * a.rows + row;
  const float* ml = a.part_ml + 2 * at;
  float M = kLowest;
  for (int s = lane; s < count; s += 64) M = fmaxf(M, ml[2 * static_cast<size_t>(s) * a.rows]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
  float acc[E] = {}, l = 0;
#pragma unroll 4
  for (int s = wave; s < count; s += 4) {
    const size_t r = static_cast<size_t>(s) * a.rows;
    const float w = exp2_fast(ml[2 * r] - M);
    l += w * ml[2 * r + 1];
    const float* p = a.part_o + (at + r) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += w * p[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) obuf[wave][lane * E + e] = acc[e];
  if (lane == 0) lbuf[wave] = l;
  __syncthreads();
  l = lbuf[0] + lbuf[1] + lbuf[2] + lbuf[3];
  if (a.final_ml && threadIdx.x == 0) {
    const size_t f = static_cast<size_t>(bh) * a.rows + row;
    a.final_ml[2 * f] = M;
    a.final_ml[2 * f + 1] = l;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int j = row / a.group, heads = a.group * a.kv.kv_heads;
  uint32_t* y = reinterpret_cast<uint32_t*>(a.out) +
                ((static_cast<size_t>(b) * a.new_tokens + j) * heads + h * a.group + row - j * a.group) *
                    (D / 2);
  const int d = 2 * threadIdx.x;
  if (d < D) {
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v[e] = (obuf[0][d + e] + obuf[1][d + e] + (obuf[2][d + e] + obuf[3][d + e])) * inv;
    y[threadIdx.x] = T::pack(v[0], v[1]);
  }
}

// weights[t] (+)= sum over rows of 2^(score - M) / l.
__global__ __launch_bounds__(256) void paged_weights_kernel(const DecodeArgs a, float* weights,
                                                            int add) {
  const int bh = blockIdx.y, b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;
  const int length = a.kv.uniform_length(b), first = length - a.new_tokens;
  const PagedTiles tiles(length, first, length - 1, a.window, a.sinks, kTileShift);
  const int P = 1 << a.kv.page_shift;
  for (int t = blockIdx.x * 256 + threadIdx.x; t < length; t += gridDim.x * 256) {
    const int page = a.kv.page(b, t >> a.kv.page_shift);
    if (page < 0) continue;
    const int tile = t >> kTileShift;
    float w = 0;
    if ((tile < tiles.sink_tiles || tile >= tiles.sink_tiles + tiles.from) &&
        ((tile + 1) << kTileShift) <= a.score_pitch) {
      const float* sp = a.scores + static_cast<size_t>(bh) * a.rows * a.score_pitch + t;
      const float* ml = a.final_ml + 2 * static_cast<size_t>(bh) * a.rows;
#pragma unroll 4
      for (int r = 0; r < a.rows; ++r) {
        const float l = ml[2 * r + 1];
        w += exp2_fast(sp[static_cast<size_t>(r) * a.score_pitch] - ml[2 * r]) *
             (l == 0.0f ? 0.0f : 1.0f / l);
      }
    }
    float* dst = weights + (static_cast<size_t>(page) * a.kv.kv_heads + h) * P + (t & (P - 1));
    *dst = add ? *dst + w : w;
  }
}

// How a call is cut: waves per row tile, splits, tiles a split takes at least.
struct DecodePlan {
  int rows, rt, zrows, splits, least, score_pitch;
  size_t o_bytes, ml_bytes, final_bytes, score_bytes;
  size_t bytes() const { return o_bytes + ml_bytes + final_bytes + score_bytes; }
};

DecodePlan plan_of(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int new_tokens, int mode) {
  DecodePlan p;
  p.rows = new_tokens * (q->heads / kv->kv_heads);
  const int row_tiles = (p.rows + 15) / 16;
  p.rt = row_tiles > 2 ? 4 : row_tiles;
  p.zrows = (row_tiles + p.rt - 1) / p.rt;
  const int len = expected_len(kv, q->max_len), window = window_of(q);
  long long tiles = (len + kTile - 1) / kTile;
  if (window > 0) {
    const long long near = (static_cast<long long>(window) + new_tokens + kTile - 2) / kTile + 1 +
                           (sinks_of(q) + kTile - 1) / kTile;
    tiles = near < tiles ? near : tiles;
  }
  const int unit = 4 / p.rt;
  const long long groups = static_cast<long long>(kv->batch) * kv->kv_heads * p.zrows;
  const long long most = (tiles + unit - 1) / unit;
  long long want = (8LL * cu_count() + groups - 1) / groups;
  want = want < most ? want : most;
  p.splits = static_cast<int>(want < 1 ? 1 : want);
  p.least = static_cast<int>((tiles + p.splits - 1) / p.splits);
  p.least = (p.least + unit - 1) / unit * unit;
  p.splits = static_cast<int>((tiles + p.least - 1) / p.least);
  if (p.splits < 1) p.splits = 1;
  const size_t bh = static_cast<size_t>(kv->batch) * kv->kv_heads, parts = bh * p.splits * p.rows;
  p.o_bytes = p.splits > 1 ? parts * kv->head_dim * 4 : 0;
  p.ml_bytes = p.splits > 1 ? parts * 8 : 0;
  p.score_pitch = mode ? (len + kTile - 1) / kTile * kTile : 0;
  p.final_bytes = mode ? (bh * p.rows * 8 + 15) / 16 * 16 : 0;
  p.ml_bytes = (p.ml_bytes + 15) / 16 * 16;
  p.score_bytes = mode ? bh * p.rows * p.score_pitch * 4 : 0;
  return p;
}

template <typename T, int D>
int launch(const DecodeArgs& a, const DecodePlan& p, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(static_cast<long long>(a.kv.batch) * a.kv.kv_heads *
                                              p.zrows * p.splits);
  if (p.rt == 1)
    paged_decode_kernel<T, D, 1><<<grid, 256, 0, stream>>>(a);
  else if (p.rt == 2)
    paged_decode_kernel<T, D, 2><<<grid, 256, 0, stream>>>(a);
  else
    paged_decode_kernel<T, D, 4><<<grid, 256, 0, stream>>>(a);
  if (p.splits > 1) {
    if (const int rc = launch_status()) return rc;
    paged_join_kernel<T, D><<<a.kv.batch * a.kv.kv_heads * a.rows, 256, 0, stream>>>(a, 4 / p.rt);
  }
  return launch_status();
}

template <typename T>
int launch_d(int D, const DecodeArgs& a, const DecodePlan& p, hipStream_t stream) {
  return D == 64    ? launch<T, 64>(a, p, stream)
         : D == 128 ? launch<T, 128>(a, p, stream)
                    : launch<T, 256>(a, p, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, int new_tokens, int mode) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (new_tokens < 1 || mode < 0 || mode > CUDALM_PAGED_WEIGHTS_ADD) return CUDALM_W4A16_EINVAL;
  if (static_cast<long long>(new_tokens) * (q->heads / kv->kv_heads) > 1024)
    return CUDALM_W4A16_EINVAL;
  const DecodePlan p = plan_of(kv, q, new_tokens, mode);
  const long long bh = static_cast<long long>(kv->batch) * kv->kv_heads;
  if (bh * p.zrows * p.splits >= kMaxGemmTiles || bh * p.rows >= kMaxGemmTiles ||
      (mode && bh > 65535))
    return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

}  // namespace

int paged_decode_regs(int type, int D) {
  if (type == CUDALM_PAGED_BF16)
    return D == 64    ? regs_of(paged_decode_kernel<PagedBf16, 64, 1>)
           : D == 128 ? regs_of(paged_decode_kernel<PagedBf16, 128, 1>)
           : D == 256 ? regs_of(paged_decode_kernel<PagedBf16, 256, 1>)
                      : -1;
  return D == 64    ? regs_of(paged_decode_kernel<PagedF16, 64, 1>)
         : D == 128 ? regs_of(paged_decode_kernel<PagedF16, 128, 1>)
         : D == 256 ? regs_of(paged_decode_kernel<PagedF16, 256, 1>)
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
  if (p.splits > 1) {
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
  a.splits = p.splits;
  a.least = p.least;
  a.window = window_of(q);
  a.sinks = sinks_of(q);
  a.score_pitch = p.score_pitch;
  const int rc = kv->type == CUDALM_PAGED_BF16 ? launch_d<PagedBf16>(kv->head_dim, a, p, stream)
                                               : launch_d<PagedF16>(kv->head_dim, a, p, stream);
  if (rc || !weights_mode) return rc;
  const dim3 grid((p.score_pitch + 255) / 256, kv->batch * kv->kv_heads);
  paged_weights_kernel<<<grid, 256, 0, stream>>>(a, kv->weights,
                                                 weights_mode == CUDALM_PAGED_WEIGHTS_ADD);
  return launch_status();
}
