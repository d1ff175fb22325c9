// The paged cache itself: argument checks, writing new tokens, eviction.

#include "paged_device.h"

namespace cudalm_hip {

int paged_check(const cudalm_paged_kv* kv) {
  if (!kv) return CUDALM_W4A16_ENULL;
  const int P = kv->page_size, D = kv->head_dim;
  if (kv->num_pages < 1 || kv->kv_heads < 1 || kv->batch < 1 || kv->max_pages < 1 || P < 16 ||
      P > 1024 || (P & (P - 1)) || (D != 64 && D != 128 && D != 256) ||
      (kv->type != CUDALM_PAGED_BF16 && kv->type != CUDALM_PAGED_F16))
    return CUDALM_W4A16_EINVAL;
  if (!kv->k || !kv->v || !kv->tables || !kv->lens) return CUDALM_W4A16_ENULL;
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->weights, 4) ||
      !aligned(kv->tables, 4) || !aligned(kv->lens, 4))
    return CUDALM_W4A16_EALIGN;
  // positions are held in 30 bits, (sequence, head) pairs in 24
  if (static_cast<long long>(kv->max_pages) * P > (1 << 30) ||
      static_cast<long long>(kv->batch) * kv->kv_heads > (1 << 24))
    return CUDALM_W4A16_ERANGE;
  return CUDALM_W4A16_OK;
}

int paged_check_query(const cudalm_paged_kv* kv, const cudalm_paged_query* q) {
  if (const int rc = paged_check(kv)) return rc;
  if (!q) return CUDALM_W4A16_ENULL;
  if (q->heads < 1 || q->heads % kv->kv_heads || q->heads / kv->kv_heads > 64)
    return CUDALM_W4A16_EINVAL;
  if (q->token_stride % 8 || q->head_stride % 8 || !aligned(q->q, 16) || !aligned(q->out, 16))
    return CUDALM_W4A16_EALIGN;
  return CUDALM_W4A16_OK;
}

namespace {

struct AppendArgs {
  PagedView kv;
  uint16_t* ck;
  uint16_t* cv;
  float* weights;
  const uint16_t* k;
  const uint16_t* v;
  long long k_token, k_head, v_token, v_head;
  const int32_t* cu;
  int tokens, each;  // each: new tokens of every sequence where cu is NULL
};

// One workgroup per eight positions (aligned: one interleaved group of V) of a
// sequence and head. A sequence of n new tokens touches at most n / 8 + 2 such
// groups, so group g of sequence b is unit cu[b] / 8 + 2 b + g, and no prefix
// sum of the group counts is needed. Eight tokens' keys are rows to copy; their
// values are read a channel pair of each token at a time and written as whole
// 16-byte units, or, where the group is only partly new, element by element,
// since its other tokens are not this call's. Bound by bytes for prompts (8 of up to
// 2001 tokens, 8 heads of 128, 88 MB: 22 us, 4.0 TB/s) and by latency for a
// decode step (32 sequences: 3 us).
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
  const int h = blockIdx.y;
  int b, begin, n, g;
  if (a.cu) {
    b = sequence_of(a.cu, a.kv.batch, blockIdx.x, 1, 8, 2);
    if (b < 0) return;
    begin = a.cu[b];
    const int end = a.cu[b + 1];
    n = begin >= 0 && end > begin ? end - begin : 0;
    g = static_cast<int>(blockIdx.x) - (begin / 8 + 2 * b);
  } else {
    const int units = a.each / 8 + 2;
    b = blockIdx.x / units;
    begin = b * a.each;
    n = a.each;
    g = blockIdx.x % units;
  }
  if (n < 1 || n > a.tokens - begin || g < 0) return;  // (g < 0 where cu does not ascend)
  const int length = a.kv.length(b), first = length - n;  // position of row `begin`
  const int p0 = (((first > 0 ? first : 0) >> 3) + g) * 8;
  if (p0 >= length) return;
  const int page = a.kv.page(b, p0 >> a.kv.page_shift);
  if (page < 0) return;
  const int P = 1 << a.kv.page_shift, off = p0 & (P - 1);
  const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + h;
  const int lo = first > p0 ? first - p0 : 0, hi = length - p0 < 8 ? length - p0 : 8;
  const long long row0 = static_cast<long long>(begin) + p0 - first;  // of token 0 of the group
  uint16_t* ck = a.ck + (head * P + off) * D;
  uint16_t* cv = a.cv + (head * P + off) * D;
  if (a.weights && threadIdx.x >= lo && threadIdx.x < hi)
    a.weights[head * P + off + threadIdx.x] = 0.0f;
  for (int i = threadIdx.x; i < D; i += 256) {
    const int c = i % (D / 8), t = i / (D / 8);
    if (t >= lo && t < hi)
      *reinterpret_cast<u32x4_t*>(ck + t * D + 8 * c) = *reinterpret_cast<const u32x4_t*>(
          a.k + (row0 + t) * a.k_token + h * a.k_head + 8 * c);
  }
  const int d = 2 * threadIdx.x;
  if (d >= D) return;
  uint32_t pair[8];
#pragma unroll
  for (int t = 0; t < 8; ++t)
    if (t >= lo && t < hi)
      pair[t] = *reinterpret_cast<const uint32_t*>(a.v + (row0 + t) * a.v_token + h * a.v_head + d);
  if (lo == 0 && hi == 8) {
    u32x4_t even, odd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      even[i] = (pair[2 * i] & 0xFFFFu) | (pair[2 * i + 1] << 16);
      odd[i] = (pair[2 * i] >> 16) | (pair[2 * i + 1] & 0xFFFF0000u);
    }
    *reinterpret_cast<u32x4_t*>(cv + 8 * d) = even;
    *reinterpret_cast<u32x4_t*>(cv + 8 * d + 8) = odd;
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (t >= lo && t < hi) {
        cv[8 * d + t] = static_cast<uint16_t>(pair[t]);
        cv[8 * d + 8 + t] = static_cast<uint16_t>(pair[t] >> 16);
      }
  }
}

struct EvictArgs {
  PagedView kv;
  uint16_t* ck;
  uint16_t* cv;
  float* weights;
  const int32_t* dst;
  int32_t* kept;      // [batch][kv_heads][keep]
  int32_t* new_lens;  // [batch]
  uint32_t* keys;     // [batch * kv_heads][pitch]
  int dst_pages, keep, sinks, recent, lds_keys;
  long long pitch;
};

// A weight's rank as a whole number: NaN lowest (1), -0 as +0; 0 stands for absent
// tokens, all ones for the first and last ones, which stay.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  return w != w ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelect = 1024;             // threads of a selecting workgroup
constexpr int kSelectLdsKeys = 32 * 1024;  // keys that it holds in LDS at most
constexpr int kSelectWords = 320;          // before the keys in LDS

// Adds 1 to hist[digit] for every lane with `in`: those that share the first one's
// digit at once, since weights of one magnitude (or all zero) share their upper
// digits, the others each.
__device__ __forceinline__ void count_digit(uint32_t* hist, uint32_t digit, bool in) {
  const uint64_t some = __ballot(in);
  if (!some) return;
  const int leader = __builtin_ctzll(some);
  const bool same = in && digit == static_cast<uint32_t>(__builtin_amdgcn_readlane(digit, leader));
  const uint64_t all = __ballot(same);
  if (in && !same) atomicAdd(&hist[digit], 1u);
  if ((threadIdx.x & 63) == static_cast<unsigned>(leader))
    atomicAdd(&hist[digit], static_cast<uint32_t>(__popcll(all)));
}

// One workgroup per (sequence, head): the key of the keep-th token in the order of
// the keys, eight bits a pass over a histogram, then the kept positions in order:
// each wave takes a sixteenth of the sequence, counts, and writes from where the
// waves before it end. The keys are made once (weights four at a time through the
// tables) and held in LDS, those of longer sequences in the workspace. Bound by the
// chain of passes of one workgroup: four chats of up to 4096 tokens 11 us, 12 documents
// of up to 30000 46 us (75 with keys in the workspace, one weight per load, and an
// atomic per key).
__global__ __launch_bounds__(kSelect) void paged_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t select_lds[];
  uint32_t* hist = select_lds;
  uint32_t* found = hist + 256;  // digit, tokens with larger keys
  uint32_t* above = found + 4;   // of each wave
  uint32_t* equal = above + kSelect / 64;
  static_assert(260 + 2 * (kSelect / 64) <= kSelectWords, "");
  const int bh = blockIdx.x, b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int length = a.kv.length(b);
  uint32_t* keys = length <= a.lds_keys ? select_lds + kSelectWords : a.keys + bh * a.pitch;
  const int s = a.sinks < a.keep ? a.sinks : a.keep;
  const int r = a.recent < a.keep - s ? a.recent : a.keep - s;
  const int P = 1 << a.kv.page_shift;
#pragma unroll 4
  for (int t = 4 * tid; t < length; t += 4 * kSelect) {
    const int page = a.kv.page(b, t >> a.kv.page_shift);
    typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
    const f32x4_any_t w = *reinterpret_cast<const f32x4_any_t*>(
        a.weights + (static_cast<size_t>(page < 0 ? 0 : page) * a.kv.kv_heads + h) * P + (t & (P - 1)));
    u32x4_t k = {weight_key(w[0]), weight_key(w[1]), weight_key(w[2]), weight_key(w[3])};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t + i < s || t + i >= length - r) k[i] = 0xFFFFFFFFu;
      if (page < 0) k[i] = 0;
    }
    *reinterpret_cast<u32x4_t*>(keys + t) = k;  // (both have room to a multiple of four)
  }
  // Ranks from the largest: the keep-th, or the last where there are fewer.
  uint32_t prefix = 0, mask = 0;
  int left = a.keep;  // rank of the wanted key among those that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t0 = 4 * (tid - lane); t0 < length; t0 += 4 * kSelect) {
      const int t = t0 + 4 * lane;
      u32x4_t k = {0, 0, 0, 0};
      if (t < length) k = *reinterpret_cast<const u32x4_t*>(keys + t);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        count_digit(hist, (k[i] >> shift) & 255, t + i < length && (k[i] & mask) == prefix);
    }
    __syncthreads();
    if (tid < 64) {
      // lane i sums digits 255 - 4 i .. 252 - 4 i, then the digits above
      uint32_t c[4], sum = 0;
      for (int i = 0; i < 4; ++i) sum += c[i] = hist[255 - 4 * lane - i];
      uint32_t incl = sum;
      for (int x = 1; x < 64; x <<= 1) {
        const uint32_t o = __shfl_up(incl, x);
        if (lane >= x) incl += o;
      }
      const uint32_t total = __shfl(incl, 63);
      uint32_t before = incl - sum;
      const uint32_t want = static_cast<uint32_t>(left) < total ? left : total;
      if (total == 0) {
        if (lane == 0) found[0] = 0, found[1] = 0;
      } else if (before < want && incl >= want) {
        for (int i = 0; i < 4; ++i) {
          if (before + c[i] >= want) {
            found[0] = 255 - 4 * lane - i;
            found[1] = before;
            break;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= 255u << shift;
    left -= static_cast<int>(found[1]);
  }
  // tokens with larger keys stay, and the first `left` of those that have this
  // one (none with key 0: absent)
  const uint32_t key = prefix;
  const int part = ((length + kSelect - 1) / kSelect) * 64;  // positions per wave
  const int t0 = wave * part, t1 = t0 + part < length ? t0 + part : length;
  int na = 0, ne = 0;
  for (int t = t0; t < t1; t += 64) {
    const uint32_t k = t + lane < t1 ? keys[t + lane] : 0;
    na += __popcll(__ballot(k > key));
    ne += __popcll(__ballot(k == key && k != 0 && t + lane < t1));
  }
  if (lane == 0) above[wave] = na, equal[wave] = ne;
  __syncthreads();
  int at = 0, eq = 0, all = 0, alleq = 0;
  for (int w = 0; w < kSelect / 64; ++w) {
    if (w < wave) at += above[w], eq += equal[w];
    all += above[w];
    alleq += equal[w];
  }
  const int ties = left < alleq ? left : alleq;
  at += eq < ties ? eq : ties;
  int32_t* kept = a.kept + static_cast<size_t>(bh) * a.keep;
  for (int t = t0; t < t1; t += 64) {
    const uint32_t k = t + lane < t1 ? keys[t + lane] : 0;
    const uint64_t e = __ballot(k == key && k != 0 && t + lane < t1);
    const uint64_t below = (1ull << lane) - 1;
    const bool stays = k > key || (((e >> lane) & 1) && eq + __popcll(e & below) < ties);
    const uint64_t st = __ballot(stays);
    if (stays) {
      const int i = at + __popcll(st & below);
      if (i < a.keep) kept[i] = t + lane;
    }
    at += __popcll(st);
    eq += __popcll(e);
  }
  const int count = all + ties < a.keep ? all + ties : a.keep;
  for (int i = count + tid; i < a.keep; i += kSelect) kept[i] = -1;
}

constexpr int kMove = 32;  // kept tokens of a copying workgroup

// 32 kept tokens of a (sequence, head) per workgroup: their places first, a thread
// each, so that the chain kept position, page, address is walked once for all; then
// their key rows, and eight tokens' values of a channel per thread, one interleaved
// unit of the fresh page. Bound by bytes: every line of the old values that holds a
// kept token is read, which for a quarter kept is nine in ten. 12 x 8 heads cut from
// up to 30000 to 8000 tokens: 195-214 us (card to card); counters show 711 MB fetched and
// 396 written, 5.2 TB/s, a copy's rate. (A thread per place took 413.)
template <int D>
__global__ __launch_bounds__(256) void paged_compact_kernel(const EvictArgs a) {
  __shared__ long long src[kMove];  // place in the cache, in tokens; -1: none
  __shared__ long long dst[kMove];
  const int tid = threadIdx.x;
  const int bh = blockIdx.y, b = bh / a.kv.kv_heads, h = bh % a.kv.kv_heads;
  const int i0 = blockIdx.x * kMove;
  const int P = 1 << a.kv.page_shift;
  if (tid < kMove) {
    const int32_t* kept = a.kept + static_cast<size_t>(bh) * a.keep;
    const int i = i0 + tid, pos = i < a.keep ? kept[i] : -1;
    // The new length here and not in the selection: there, new_lens may be the lengths
    // that other heads' workgroups have still to read. It is where kept ends.
    if (h == 0) {
      if (pos >= 0 && (i + 1 == a.keep || kept[i + 1] < 0)) a.new_lens[b] = i + 1;
      if (i == 0 && pos < 0) a.new_lens[b] = 0;
    }
    const int pi = i >> a.kv.page_shift;
    const int to = pi < a.dst_pages ? a.dst[static_cast<size_t>(b) * a.dst_pages + pi] : -1;
    const int from = pos >= 0 ? a.kv.page(b, pos >> a.kv.page_shift) : -1;
    long long s = -1, d = -1;
    if (from >= 0 && to >= 0 && to < a.kv.num_pages) {
      s = (static_cast<long long>(from) * a.kv.kv_heads + h) * P + (pos & (P - 1));
      d = (static_cast<long long>(to) * a.kv.kv_heads + h) * P + (i & (P - 1));
      a.weights[d] = a.weights[s];
    }
    src[tid] = s;
    dst[tid] = d;
  }
  __syncthreads();
  constexpr int C = D / 8;
#pragma unroll 4
  for (int u = tid; u < kMove * C; u += 256) {
    const int t = u / C, c = u % C;
    const long long s = src[t];
    if (s >= 0)
      *reinterpret_cast<u32x4_t*>(a.ck + dst[t] * D + 8 * c) =
          *reinterpret_cast<const u32x4_t*>(a.ck + s * D + 8 * c);
  }
#pragma unroll 4
  for (int u = tid; u < kMove / 8 * D; u += 256) {
    const int g = u / D * 8, d = u % D;
    uint32_t x[8];
    bool all = true;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const long long s = src[g + t];
      all = all && s >= 0;
      x[t] = s >= 0 ? a.cv[(s & ~7LL) * D + 8 * d + (s & 7)] : 0;
    }
    if (all) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[2 * i] | (x[2 * i + 1] << 16);
      *reinterpret_cast<u32x4_t*>(a.cv + dst[g] * D + 8 * d) = w;
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (src[g + t] >= 0)
          a.cv[(dst[g + t] & ~7LL) * D + 8 * d + t] = static_cast<uint16_t>(x[t]);
    }
  }
}

}  // namespace

int paged_decode_regs(int type, int D);
int paged_prefill_regs(int type, int D);

}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" int cudalm_paged_append(const cudalm_paged_kv* kv, const void* k, const void* v,
                                   int64_t k_token_stride, int64_t k_head_stride,
                                   int64_t v_token_stride, int64_t v_head_stride,
                                   const int32_t* cu_new, int tokens, hipStream_t stream) {
  if (const int rc = paged_check(kv)) return rc;
  if (tokens < 0 || (!cu_new && tokens % kv->batch)) return CUDALM_W4A16_EINVAL;
  if (tokens == 0) return CUDALM_W4A16_OK;
  if (!k || !v) return CUDALM_W4A16_ENULL;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(cu_new, 4) || k_token_stride % 8 ||
      k_head_stride % 8 || v_token_stride % 8 || v_head_stride % 8)
    return CUDALM_W4A16_EALIGN;
  const long long units = cu_new ? static_cast<long long>(tokens) / 8 + 2LL * kv->batch
                                 : static_cast<long long>(kv->batch) *
                                       (tokens / kv->batch / 8 + 2);
  if (units >= kMaxGemmTiles || kv->kv_heads > 65535 || units * kv->kv_heads >= kMaxGemmTiles)
    return CUDALM_W4A16_ERANGE;
  AppendArgs a = {view_of(kv),
                  static_cast<uint16_t*>(kv->k),
                  static_cast<uint16_t*>(kv->v),
                  kv->weights,
                  static_cast<const uint16_t*>(k),
                  static_cast<const uint16_t*>(v),
                  k_token_stride,
                  k_head_stride,
                  v_token_stride,
                  v_head_stride,
                  cu_new,
                  tokens,
                  cu_new ? 0 : tokens / kv->batch};
  const dim3 grid(static_cast<unsigned>(units), kv->kv_heads);
  if (kv->head_dim == 64)
    paged_append_kernel<64><<<grid, 256, 0, stream>>>(a);
  else if (kv->head_dim == 128)
    paged_append_kernel<128><<<grid, 256, 0, stream>>>(a);
  else
    paged_append_kernel<256><<<grid, 256, 0, stream>>>(a);
  return launch_status();
}

extern "C" size_t cudalm_paged_evict_workspace_bytes(const cudalm_paged_kv* kv, int max_len) {
  if (paged_check(kv) != CUDALM_W4A16_OK) return 0;
  (void)max_len;
  return static_cast<size_t>(kv->batch) * kv->kv_heads * kv->max_pages * kv->page_size * 4;
}

extern "C" int cudalm_paged_evict(const cudalm_paged_kv* kv, const int32_t* dst_tables,
                                  int dst_pages, int keep, int sinks, int recent, int32_t* kept,
                                  int32_t* new_lens, int max_len, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = paged_check(kv)) return rc;
  if (keep < 1 || sinks < 0 || recent < 0 || dst_pages < 1 ||
      static_cast<long long>(dst_pages) * kv->page_size < keep)
    return CUDALM_W4A16_EINVAL;
  if (!kv->weights || !dst_tables || !kept || !new_lens || !workspace) return CUDALM_W4A16_ENULL;
  if (!aligned(dst_tables, 4) || !aligned(kept, 4) || !aligned(new_lens, 4) ||
      !aligned(workspace, 16))
    return CUDALM_W4A16_EALIGN;
  const long long bh = static_cast<long long>(kv->batch) * kv->kv_heads;
  const long long groups = (static_cast<long long>(keep) + kMove - 1) / kMove;
  if (workspace_bytes < cudalm_paged_evict_workspace_bytes(kv, max_len) || bh > 65535 ||
      groups * bh >= kMaxGemmTiles)
    return CUDALM_W4A16_ERANGE;
  EvictArgs a = {view_of(kv),
                 static_cast<uint16_t*>(kv->k),
                 static_cast<uint16_t*>(kv->v),
                 kv->weights,
                 dst_tables,
                 kept,
                 new_lens,
                 static_cast<uint32_t*>(workspace),
                 dst_pages,
                 keep,
                 sinks,
                 recent,
                 0,
                 static_cast<long long>(kv->max_pages) * kv->page_size};
  const int expected = (expected_len(kv, max_len) + 3) / 4 * 4;
  a.lds_keys = expected < kSelectLdsKeys ? expected : kSelectLdsKeys;
  if (!allow_lds(paged_select_kernel, 4 * (kSelectWords + kSelectLdsKeys))) return CUDALM_W4A16_ELAUNCH;
  paged_select_kernel<<<static_cast<unsigned>(bh), kSelect, 4 * (kSelectWords + a.lds_keys),
                        stream>>>(a);
  if (const int rc = launch_status()) return rc;
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(bh));
  if (kv->head_dim == 64)
    paged_compact_kernel<64><<<grid, 256, 0, stream>>>(a);
  else if (kv->head_dim == 128)
    paged_compact_kernel<128><<<grid, 256, 0, stream>>>(a);
  else
    paged_compact_kernel<256><<<grid, 256, 0, stream>>>(a);
  return launch_status();
}

extern "C" int cudalm_paged_kernel_regs(int type, int head_dim, int prefill) {
  if (type != CUDALM_PAGED_BF16 && type != CUDALM_PAGED_F16) return -1;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -1;
  return prefill ? paged_prefill_regs(type, head_dim) : paged_decode_regs(type, head_dim);
}
