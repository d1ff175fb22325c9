// Attention of one or a few new tokens of every sequence, where groups of sequences
// begin with the same tokens.
//
// A group's queries, those of all its sequences, are the rows of one product over its
// shared tokens (prefill's tiles, positions row by row), so a shared key or value is
// fetched once for 128 of them. Every sequence's own tokens are decode's. Both leave
// sums under a running maximum in parts, which a last kernel joins:
//
//   out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s     over the parts of both kinds

#include "paged_decode_body.h"
#include "paged_prefill_body.h"

namespace cudalm_hip {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : D == 128 ? 3 : 4) void paged_prefix_kernel(const PrefixArgs a) {
  extern __shared__ uint16_t lds[];
  paged_prefill_body<T, D>(a, lds, blockIdx.x);
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(256, 2) void paged_own_kernel(const OwnDecodeArgs a) {
  __shared__ DecodeLds<D, RT, 4> lds;
  paged_decode_body<T, D, RT, 4, true>(a, lds, blockIdx.x);
}

// A workgroup of four waves per row, a quarter of its parts each: out = the join.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_shared_join_kernel(const OwnDecodeArgs a, const float* prefix_o,
                                                                const float* prefix_ml, int splits) {
  constexpr int E = D / 64;
  __shared__ float sums[4][D], weights[4];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int heads = a.group * a.kv.kv_heads;
  const size_t rows = static_cast<size_t>(a.kv.batch) * a.new_tokens * heads, row = blockIdx.x;
  const int token = static_cast<int>(row / heads), head = static_cast<int>(row - static_cast<size_t>(token) * heads);
  const int b = token / a.new_tokens, h = head / a.group;
  const int r = (token - b * a.new_tokens) * a.group + head - h * a.group, zr = r / a.part_rows;
  const Parts own(a, b, h, zr, lane);
  const int before = uniform(a.sharing.shared_of(a.kv, b)) > 0 ? splits : 0, count = before + own.count;
  auto ml = [&](int s) {
    return s < before ? prefix_ml + 2 * (s * rows + row)
                      : a.part_ml + 2 * (own.at(s - before) * a.part_rows + r - zr * a.part_rows);
  };
  float M = kLowest;
  for (int s = lane; s < count; s += 64) M = fmaxf(M, ml(s)[0]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
  float acc[E] = {}, l = 0;
#pragma unroll 4
  for (int s = wave; s < count; s += 4) {
    const float* at = ml(s);
    const float m = at[0];
    if (m == -__builtin_inff()) continue;  // nothing to read (prefill's parts say so)
    const float w = exp2_fast(m - M);
    l += w * at[1];
    const float* p = (s < before ? prefix_o + (s * rows + row) * D
                                 : a.part_o + (own.at(s - before) * a.part_rows + r - zr * a.part_rows) * D) + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += joined(w, p[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sums[wave][lane * E + e] = acc[e];
  if (lane == 0) weights[wave] = l;
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  l = weights[0] + weights[1] + weights[2] + weights[3];
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  float y[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int c = 2 * threadIdx.x + e;
    const float v = sums[0][c] + sums[1][c] + sums[2][c] + sums[3][c];
    y[e] = l == 0.0f ? 0.0f : v * inv;  // (no weight at all: zeros, whatever the values)
  }
  reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row * D)[threadIdx.x] = T::pack(y[0], y[1]);
}

// How a call is cut.
struct SharedPlan {
  int rows, rt, zrows, part_rows, groups, least, splits;
  long long units, segments;
  size_t prefix_o, prefix_ml, own_o, own_ml;
  size_t bytes() const { return prefix_o + prefix_ml + own_o + own_ml; }
};

SharedPlan plan_of(const cudalm_paged_kv* kv, const cudalm_paged_query* q, const cudalm_paged_groups* g,
                   int new_tokens) {
  SharedPlan p;
  const int group = q->heads / kv->kv_heads;
  p.rows = new_tokens * group;
  const int row_tiles = (p.rows + 15) / 16;
  p.rt = row_tiles > 2 ? 4 : row_tiles;
  p.zrows = (row_tiles + p.rt - 1) / p.rt;
  p.part_rows = 16 * p.rt < p.rows ? 16 * p.rt : p.rows;
  p.least = 4 / p.rt;
  p.groups = (kv->head_dim == 64 ? 4 : 2) * cu_count();
  p.segments = static_cast<long long>(kv->batch) * kv->kv_heads * p.zrows;
  const size_t slots = (2 * static_cast<size_t>(p.groups) + p.segments) * p.part_rows;
  p.own_o = slots * kv->head_dim * 4;
  p.own_ml = (slots * 8 + 15) / 16 * 16;
  // the prefixes: enough workgroups to fill the chip, of at least four tiles
  const long long total = static_cast<long long>(kv->batch) * new_tokens * q->heads;
  p.units = static_cast<long long>(kv->batch) * p.rows / kRows + g->count;
  const int len = expected_len(kv, g->max_shared);
  long long tiles = (len + kTile - 1) / kTile;
  const long long groups = (static_cast<long long>(kv->batch) * p.rows + kRows - 1) / kRows * kv->kv_heads;
  long long want = 2LL * cu_count() / groups;
  want = want < tiles / 4 ? want : tiles / 4;
  want = want < 32 ? want : 32;
  p.splits = static_cast<int>(want < 1 ? 1 : want);
  p.prefix_o = static_cast<size_t>(p.splits) * total * kv->head_dim * 4;
  p.prefix_ml = (static_cast<size_t>(p.splits) * total * 8 + 15) / 16 * 16;
  return p;
}

template <typename T, int D>
int launch(const PrefixArgs& a, const OwnDecodeArgs& o, const SharedPlan& p, hipStream_t stream) {
  auto prefix = paged_prefix_kernel<T, D>;
  if (!allow_lds(prefix, kPrefillLds<D>)) return CUDALM_W4A16_ELAUNCH;
  prefix<<<static_cast<unsigned>(p.units * a.kv.kv_heads * a.splits), 64 * kWaves, kPrefillLds<D>, stream>>>(a);
  if (const int rc = launch_status()) return rc;
  auto own = p.rt == 1 ? paged_own_kernel<T, D, 1> : p.rt == 2 ? paged_own_kernel<T, D, 2> : paged_own_kernel<T, D, 4>;
  own<<<p.groups, 256, 0, stream>>>(o);
  if (const int rc = launch_status()) return rc;
  const unsigned rows = static_cast<unsigned>(a.tokens) * a.heads;
  paged_shared_join_kernel<T, D><<<rows, 256, 0, stream>>>(o, a.part_o, a.part_ml, a.splits);
  return launch_status();
}

template <typename T>
int launch_d(int D, const PrefixArgs& a, const OwnDecodeArgs& o, const SharedPlan& p, hipStream_t stream) {
  return D == 64    ? launch<T, 64>(a, o, p, stream)
         : D == 128 ? launch<T, 128>(a, o, p, stream)
                    : launch<T, 256>(a, o, p, stream);
}

int check(const cudalm_paged_kv* kv, const cudalm_paged_query* q, const cudalm_paged_groups* g, int new_tokens) {
  if (const int rc = paged_check_query(kv, q)) return rc;
  if (!g) return CUDALM_W4A16_ENULL;
  if (new_tokens < 1 || g->count < 1) return CUDALM_W4A16_EINVAL;
  if (static_cast<long long>(new_tokens) * (q->heads / kv->kv_heads) > kMaxRows) return CUDALM_W4A16_EINVAL;
  if (!g->cu || !g->shared) return CUDALM_W4A16_ENULL;
  if (!aligned(g->cu, 4) || !aligned(g->shared, 4)) return CUDALM_W4A16_EALIGN;
  const long long rows = static_cast<long long>(kv->batch) * new_tokens * q->heads;
  if (rows >= kMaxGemmTiles || g->count > kv->batch) return rows >= kMaxGemmTiles ? CUDALM_W4A16_ERANGE : CUDALM_W4A16_EINVAL;
  const SharedPlan p = plan_of(kv, q, g, new_tokens);
  // own tiles are numbered in 31 bits, and where the last workgroup's range would end
  const long long cap = (static_cast<long long>(kv->max_pages) * kv->page_size + kTile - 1) / kTile;
  const long long tiles = p.segments * (cap + 1);
  if (tiles + tiles / p.groups + p.groups >= (1LL << 31)) return CUDALM_W4A16_ERANGE;
  if (p.segments >= kMaxGemmTiles || p.units * kv->kv_heads * p.splits >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
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
  PrefixArgs a = {};
  a.kv = view_of(kv);
  a.k = static_cast<const uint16_t*>(kv->k);
  a.v = static_cast<const uint16_t*>(kv->v);
  a.q = static_cast<const uint16_t*>(q->q);
  a.out = static_cast<uint16_t*>(q->out);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + p.prefix_o);
  a.token_stride = q->token_stride;
  a.head_stride = q->head_stride;
  a.negate = q->scale < 0;
  a.scale_log2 = fmaxf((a.negate ? -q->scale : q->scale) * kLog2e, 1e-38f);  // (as in prefill)
  a.tokens = kv->batch * new_tokens;
  a.heads = q->heads;
  a.group = q->heads / kv->kv_heads;
  a.units = static_cast<int>(p.units);
  a.splits = p.splits;
  a.least = 1;
  a.window = window_of(q);
  a.sinks = sinks_of(q);
  a.sharing = {groups->cu, groups->shared, groups->count};
  a.new_tokens = new_tokens;
  OwnDecodeArgs o = {};
  o.kv = a.kv;
  o.k = a.k;
  o.v = a.v;
  o.q = a.q;
  o.out = q->out;
  o.part_o = reinterpret_cast<float*>(ws + p.prefix_o + p.prefix_ml);
  o.part_ml = reinterpret_cast<float*>(ws + p.prefix_o + p.prefix_ml + p.own_o);
  o.token_stride = q->token_stride;
  o.head_stride = q->head_stride;
  o.scale_log2 = q->scale * kLog2e;
  o.new_tokens = new_tokens;
  o.group = a.group;
  o.rows = p.rows;
  o.zrows = p.zrows;
  o.part_rows = p.part_rows;
  o.groups = p.groups;
  o.splits = 0;
  o.least = p.least;
  o.window = a.window;
  o.sinks = a.sinks;
  o.sharing = a.sharing;
  return kv->type == CUDALM_PAGED_BF16 ? launch_d<PagedBf16>(kv->head_dim, a, o, p, stream)
                                       : launch_d<PagedF16>(kv->head_dim, a, o, p, stream);
}
