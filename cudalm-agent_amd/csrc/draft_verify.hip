// Verification of drafted tokens against the target's probabilities.
//
// Probabilities become whole units of 2^-40 before they are summed, so sums are
// exact, have no order and the drawn token is the same however the vocabulary
// is split. What is read is one row of the target and one of the draft per
// sequence (where the first token is refused, or after the last), next to the
// drafted tokens' own probabilities: bytes bound a batch (64 sequences with seven
// drafted tokens of 248320, fp32, 127 MB: 22 us, 5.8 TB/s with what stays cached, and
// 9 for the draw), two launches' latency a single sequence (6 + 7 us).

#include "cudalm_draft.h"
#include "hip_common.h"

namespace cudalm_hip {
namespace {

constexpr int kChunk = 4096;  // vocabulary entries per workgroup
constexpr int kEach = kChunk / 256;
constexpr int kSumGroups = 8;  // summing workgroups per CU that run at once
constexpr int kMaxVocab = 1 << 22;  // 2^22 probabilities of at most 2^40 units: below 2^63

struct VerifyArgs {
  const void* target;
  const void* draft;
  const int32_t* tokens;
  const int32_t* counts;
  const float* u_accept;
  const float* u_next;
  int32_t* out;
  int32_t* accepted;
  uint64_t* sums;  // [batch][chunks][2]: units left over from the draft's, units of the target
  long long target_stride, draft_stride;
  int g, vocab, chunks;
};

struct ProbF32 {
  typedef float type;
  static __device__ __forceinline__ float of(u32x4_t v, int i) {
    const uint32_t x = v[i];  // (a bit cast of the element itself takes element 0)
    return __builtin_bit_cast(float, x);
  }
  static __device__ __forceinline__ float value(float x) { return x; }
};
struct ProbBf16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float of(u32x4_t v, int i) {
    return i & 1 ? bf16_hi(v[i / 2]) : bf16_lo(v[i / 2]);
  }
  static __device__ __forceinline__ float value(uint16_t x) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16);
  }
};
struct ProbF16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float of(u32x4_t v, int i) {
    return value(static_cast<uint16_t>(v[i / 2] >> (i & 1 ? 16 : 0)));
  }
  static __device__ __forceinline__ float value(uint16_t x) {
    return static_cast<float>(__builtin_bit_cast(_Float16, x));
  }
};

// Whole units of 2^-40; NaN and negative numbers are none.
__device__ __forceinline__ uint64_t units(float p) {
  return static_cast<uint64_t>(fminf(fmaxf(p, 0.0f), 1.0f) * 1099511627776.0f);
}

// The number of accepted tokens, for all threads of the workgroup.
template <typename P>
__device__ __forceinline__ int accepted_count(const VerifyArgs& a, int b, int* first_refused) {
  int n = a.counts ? a.counts[b] : a.g;
  n = n < 0 ? 0 : n < a.g ? n : a.g;
  if (threadIdx.x == 0) *first_refused = n;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int x = a.tokens[static_cast<size_t>(b) * a.g + i];
    bool accept = false;
    if (x >= 0 && x < a.vocab) {
      const float p = P::value(static_cast<const typename P::type*>(
          a.target)[(static_cast<long long>(b) * (a.g + 1) + i) * a.target_stride + x]);
      float q = 1.0f;
      if (a.draft)
        q = P::value(static_cast<const typename P::type*>(
            a.draft)[(static_cast<long long>(b) * a.g + i) * a.draft_stride + x]);
      accept = a.u_accept[static_cast<size_t>(b) * a.g + i] * q < p;
    }
    if (!accept) atomicMin(first_refused, i);
  }
  __syncthreads();
  return *first_refused;
}

// The rows the next token is drawn from: the target's, and what the draft
// takes off it (a row, or one token, or nothing).
template <typename P>
struct Rows {
  const typename P::type* p;
  const typename P::type* q;
  int one;

  __device__ __forceinline__ Rows(const VerifyArgs& a, int b, int n) {
    int count = a.counts ? a.counts[b] : a.g;
    count = count < 0 ? 0 : count < a.g ? count : a.g;
    p = static_cast<const typename P::type*>(a.target) +
        (static_cast<long long>(b) * (a.g + 1) + n) * a.target_stride;
    q = nullptr;
    one = -1;
    if (n < count) {
      if (a.draft)
        q = static_cast<const typename P::type*>(a.draft) +
            (static_cast<long long>(b) * a.g + n) * a.draft_stride;
      else
        one = a.tokens[static_cast<size_t>(b) * a.g + n];
    }
  }
  // What the draft leaves of token v's probability pv.
  __device__ __forceinline__ float left(int v, float pv, float qv) const {
    return q ? pv - qv : v == one ? pv - 1.0f : pv;
  }
  __device__ __forceinline__ float left(int v, float pv) const {
    return left(v, pv, q ? P::value(q[v]) : 0.0f);
  }
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(v), d));
}

// Inclusive prefix sum over the 256 threads; `total` gets the sum.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* waves, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int x = 1; x < 64; x <<= 1) {
    const uint64_t o = shfl_up64(v, x);
    if (lane >= x) v += o;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  uint64_t sum = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < wave) v += waves[w];
    sum += waves[w];
  }
  *total = sum;
  return v;
}

// A sequence's chunks over gridDim.x workgroups, each of which finds the number of
// accepted tokens for itself (a chain of three loads, so that no more workgroups are
// launched than run at once).
template <typename P>
__global__ __launch_bounds__(256) void draft_sum_kernel(const VerifyArgs a) {
  constexpr int V = 16 / sizeof(typename P::type);  // probabilities per load
  __shared__ int refused;
  __shared__ uint64_t waves[4];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int n = accepted_count<P>(a, b, &refused);
  // through out, and not to `accepted`, which may be the counts that other workgroups and
  // the next kernel have still to read
  if (blockIdx.x == 0 && tid == 0) a.out[static_cast<size_t>(b) * (a.g + 1)] = n;
  const Rows<P> rows(a, b, n);
  const bool wide = ((reinterpret_cast<uintptr_t>(rows.p) | reinterpret_cast<uintptr_t>(rows.q)) & 15) == 0;
  for (int chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    uint64_t rest = 0, whole = 0;
    if (wide && (chunk + 1) * kChunk <= a.vocab) {
      const u32x4_t* pp = reinterpret_cast<const u32x4_t*>(rows.p) + chunk * (kChunk / V) + tid;
      const u32x4_t* qp = reinterpret_cast<const u32x4_t*>(rows.q ? rows.q : rows.p) + chunk * (kChunk / V) + tid;
      u32x4_t p[kEach / V], q[kEach / V];
#pragma unroll
      for (int i = 0; i < kEach / V; ++i) {
        p[i] = __builtin_nontemporal_load(pp + 256 * i);
        q[i] = __builtin_nontemporal_load(qp + 256 * i);
      }
#pragma unroll
      for (int i = 0; i < kEach / V; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float pv = P::of(p[i], e);
          whole += units(pv);
          rest += units(rows.left(chunk * kChunk + (256 * i + tid) * V + e, pv, P::of(q[i], e)));
        }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int v = chunk * kChunk + tid + 256 * i;
        if (v < a.vocab) {
          const float p = P::value(rows.p[v]);
          whole += units(p);
          rest += units(rows.left(v, p));
        }
      }
    }
    uint64_t total;
    block_scan(rest, waves, &total);
    uint64_t* s = a.sums + 2 * (static_cast<size_t>(b) * a.chunks + chunk);
    if (tid == 0) s[0] = total;
    block_scan(whole, waves, &total);
    if (tid == 0) s[1] = total;
  }
}

// One workgroup per sequence: the chunk that holds the mark, then the token in it, by
// prefix sums of whole units. Latency bounds it, 7 to 9 us: the chunks' sums, two scans,
// one chunk, a scan.
template <typename P>
__global__ __launch_bounds__(256) void draft_pick_kernel(const VerifyArgs a) {
  __shared__ int chunk, token;
  __shared__ uint64_t waves[4], before;
  const int b = blockIdx.x, tid = threadIdx.x;
  int32_t* out = a.out + static_cast<size_t>(b) * (a.g + 1);
  const int n = out[0];
  const Rows<P> rows(a, b, n);
  const uint64_t* s = a.sums + 2 * static_cast<size_t>(b) * a.chunks;
  uint64_t c[2][4], sum[2] = {0, 0}, total[2];
  for (int i = 0; i < 4; ++i)
    for (int k = 0; k < 2; ++k) {
      c[k][i] = 4 * tid + i < a.chunks ? s[2 * (4 * tid + i) + k] : 0;
      sum[k] += c[k][i];
    }
  uint64_t incl[2];
  incl[0] = block_scan(sum[0], waves, &total[0]);
  incl[1] = block_scan(sum[1], waves, &total[1]);
  const int k = total[0] > 0 ? 0 : 1;
  float u = a.u_next[b] * 16777216.0f;
  u = fminf(fmaxf(u, 0.0f), 16777215.0f);
  const uint64_t U = static_cast<uint64_t>(u);
  const uint64_t mark = (total[k] >> 24) * U + (((total[k] & 0xFFFFFF) * U) >> 24);
  if (tid == 0) token = -1, chunk = -1;
  __syncthreads();
  uint64_t below = incl[k] - sum[k];
  for (int i = 0; i < 4; ++i) {
    if (below <= mark && mark < below + c[k][i]) chunk = 4 * tid + i, before = below;
    below += c[k][i];
  }
  __syncthreads();
  if (chunk >= 0) {
    uint64_t x[kEach], mine = 0, all;
    const int v0 = chunk * kChunk + tid * kEach;
    for (int i = 0; i < kEach; ++i) {
      x[i] = 0;
      if (v0 + i < a.vocab) {
        const float p = P::value(rows.p[v0 + i]);
        x[i] = units(k == 0 ? rows.left(v0 + i, p) : p);
      }
      mine += x[i];
    }
    uint64_t at = before + block_scan(mine, waves, &all) - mine;
    for (int i = 0; i < kEach; ++i) {
      if (at <= mark && mark < at + x[i]) token = v0 + i;
      at += x[i];
    }
  }
  __syncthreads();
  if (tid == 0) a.accepted[b] = n;
  for (int i = tid; i <= a.g; i += 256)
    out[i] = i < n ? a.tokens[static_cast<size_t>(b) * a.g + i] : i == n ? token : -1;
}

template <typename P>
int launch(const VerifyArgs& a, int batch, hipStream_t stream) {
  const int at_once = kSumGroups * cu_count() / batch;
  const int groups = at_once < 1 ? 1 : at_once < a.chunks ? at_once : a.chunks;
  draft_sum_kernel<P><<<dim3(groups, batch), 256, 0, stream>>>(a);
  if (const int rc = launch_status()) return rc;
  draft_pick_kernel<P><<<batch, 256, 0, stream>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" size_t cudalm_draft_verify_workspace_bytes(int batch, int draft, int vocab) {
  if (batch < 1 || batch > 65535 || draft < 0 || vocab < 1 || vocab > kMaxVocab) return 0;
  return static_cast<size_t>(batch) * ((vocab + kChunk - 1) / kChunk) * 16;
}

extern "C" int cudalm_draft_verify(const void* target, int64_t target_stride,
                                   const void* draft_probs, int64_t draft_stride, int type,
                                   const int32_t* tokens, const int32_t* counts,
                                   const float* u_accept, const float* u_next, int32_t* out,
                                   int32_t* accepted, int batch, int draft, int vocab,
                                   void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (batch < 1 || draft < 0 || vocab < 1 || type < CUDALM_DRAFT_F32 || type > CUDALM_DRAFT_F16 ||
      target_stride < vocab || (draft_probs && draft_stride < vocab))
    return CUDALM_W4A16_EINVAL;
  if (!target || !u_next || !out || !accepted || !workspace || (draft > 0 && (!tokens || !u_accept)))
    return CUDALM_W4A16_ENULL;
  const uintptr_t elem = type == CUDALM_DRAFT_F32 ? 4 : 2;
  if (!aligned(target, elem) || !aligned(draft_probs, elem) || !aligned(tokens, 4) ||
      !aligned(counts, 4) || !aligned(u_accept, 4) || !aligned(u_next, 4) || !aligned(out, 4) ||
      !aligned(accepted, 4) || !aligned(workspace, 8))
    return CUDALM_W4A16_EALIGN;
  const size_t need = cudalm_draft_verify_workspace_bytes(batch, draft, vocab);
  if (need == 0 || workspace_bytes < need || draft > (1 << 20) ||
      static_cast<long long>(batch) * ((vocab + kChunk - 1) / kChunk) >= kMaxGemmTiles)
    return CUDALM_W4A16_ERANGE;
  VerifyArgs a = {target,
                  draft > 0 ? draft_probs : nullptr,
                  tokens,
                  counts,
                  u_accept,
                  u_next,
                  out,
                  accepted,
                  static_cast<uint64_t*>(workspace),
                  target_stride,
                  draft_stride,
                  draft,
                  vocab,
                  (vocab + kChunk - 1) / kChunk};
  return type == CUDALM_DRAFT_F32    ? launch<ProbF32>(a, batch, stream)
         : type == CUDALM_DRAFT_BF16 ? launch<ProbBf16>(a, batch, stream)
                                     : launch<ProbF16>(a, batch, stream);
}
