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

#include "paged_prefill_body.h"

namespace cudalm_hip {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : D == 128 ? 3 : 4) void paged_prefill_kernel(const PrefillArgs a) {
  extern __shared__ uint16_t lds[];
  paged_prefill_body<T, D>(a, lds, blockIdx.x);
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
  if (!allow_lds(kernel, kPrefillLds<D>)) return CUDALM_W4A16_ELAUNCH;
  const unsigned grid = static_cast<unsigned>(a.units) * a.kv.kv_heads * a.splits;
  kernel<<<grid, 64 * kWaves, kPrefillLds<D>, stream>>>(a);
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
