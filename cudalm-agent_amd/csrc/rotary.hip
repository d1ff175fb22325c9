// Rotary positions: rows of heads rotated by their positions, and new tokens' keys
// rotated on their way into the pages of the paged cache.
//
// The cosines and sines of a token's pairs are those of all its heads: a workgroup takes
// up to eight tokens, makes theirs once in LDS, and every thread keeps those of eight
// pairs of one token in registers while it walks over heads. p f / pi is made in 64-bit floats
// (three roundings: 31 bits of position times 24 of frequency are two more than a double has),
// reduced there to [-1, 1], and only then rounded to fp32 for the sine. That last rounding, 2^-25, is
// the larger one up to angles of 2^27.

#include "cudalm_rotary.h"

#include "paged_device.h"
#include "row_places.h"

namespace cudalm_hip {
namespace {

constexpr int kTokens = 8;   // of a workgroup at most; a group of eight values in the cache
constexpr int kThreads = 256;

// How rows are turned. Axis of pair i: bits 2 i of `axis`.
struct Turn {
  const float* freqs;
  const int32_t* positions;  // [axes][tokens], or NULL: consecutive from the first token's
  long long tokens;
  int pairs, adjacent;
  float scale;
  uint32_t axis[CUDALM_ROTARY_MAX_PAIRS / 16];
};

// cosine and sine of `count` tokens' pairs: row `row0` on, places p0 on.
__device__ __forceinline__ void make_angles(float2* cs, const Turn& a, long long row0, int p0,
                                            int count) {
  for (int i = threadIdx.x; i < count * a.pairs; i += kThreads) {
    const int t = i / a.pairs, pair = i - t * a.pairs;
    int p = p0 + t;
    if (a.positions) {
      const int axis = (a.axis[pair >> 4] >> (2 * (pair & 15))) & 3;
      p = a.positions[axis * a.tokens + row0 + t];
    }
    const double half_turns = static_cast<double>(p) * static_cast<double>(a.freqs[pair]) *
                              0.318309886183790671537767526745;
    const float r = static_cast<float>(half_turns - 2.0 * rint(0.5 * half_turns));
    float s, c;
    sincospif(r, &s, &c);
    cs[i] = float2{c * a.scale, s * a.scale};
  }
}

// Twice eight channels of a token: eight pairs, or channels that are copied. The second
// eight are half of the rotated (copied) channels further, so that threads side by side
// have channels side by side.
struct Chunk {
  int at0, at1;      // channels; at1 < 0: none
  int pair0, pair1;  // of the first four pairs and the others
  bool turned;
};
__device__ __forceinline__ Chunk chunk_of(const Turn& a, int c, int D) {
  const int turned = a.pairs / 8;
  Chunk r;
  r.turned = c < turned;
  if (r.turned) {
    r.at0 = 8 * c;
    r.at1 = a.pairs + 8 * c;
    r.pair0 = a.adjacent ? 4 * c : 8 * c;
    r.pair1 = a.adjacent ? a.pairs / 2 + 4 * c : 8 * c + 4;
  } else {
    const int eights = (D - 2 * a.pairs) / 8, half = (eights + 1) / 2, i = c - turned;
    r.at0 = 2 * a.pairs + 8 * i;
    r.at1 = i + half < eights ? r.at0 + 8 * half : -1;
    r.pair0 = r.pair1 = 0;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void turn_pair(const float2 cs, float& x0, float& x1) {
  const float y0 = __builtin_fmaf(x0, cs.x, -(x1 * cs.y));
  x1 = __builtin_fmaf(x1, cs.x, x0 * cs.y);
  x0 = y0;
}

template <typename T>
__device__ __forceinline__ float upper(uint32_t w) {
  return T::value(static_cast<uint16_t>(w >> 16));
}
template <typename T>
__device__ __forceinline__ float lower(uint32_t w) {
  return T::value(static_cast<uint16_t>(w));
}

// Turns the pairs that u and v hold: element e of both is a pair, or those side by side.
template <typename T>
__device__ __forceinline__ void turn_chunk(bool adjacent, const float2* cs, u32x4_t& u, u32x4_t& v) {
  if (adjacent) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x0 = lower<T>(u[e]), x1 = upper<T>(u[e]);
      turn_pair<T>(cs[e], x0, x1);
      u[e] = T::pack(x0, x1);
      x0 = lower<T>(v[e]), x1 = upper<T>(v[e]);
      turn_pair<T>(cs[4 + e], x0, x1);
      v[e] = T::pack(x0, x1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x0 = lower<T>(u[e]), x1 = lower<T>(v[e]), z0 = upper<T>(u[e]), z1 = upper<T>(v[e]);
      turn_pair<T>(cs[2 * e], x0, x1);
      turn_pair<T>(cs[2 * e + 1], z0, z1);
      u[e] = T::pack(x0, z0);
      v[e] = T::pack(x1, z1);
    }
  }
}

// Results pass the caches by: nothing here reads them again (19201 rows of 16 heads of 128: 34
// us with ordinary stores, 27 so; eight prompts 63 and 58).
__device__ __forceinline__ void stream16(uint16_t* p, u32x4_t v) {
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(p));
}

// The same for what is read once (eight prompts: 56 us; rotate_kernel is the slower one with
// it, 30).
template <typename V>
__device__ __forceinline__ V load_once(const uint16_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

struct RotateArgs {
  Turn turn;
  const uint16_t* x;
  uint16_t* out;
  long long x_token, x_head, out_token, out_head;
  int heads, D, each;  // each: tokens of a workgroup
};

// 16 bytes at a time. Bytes bound it: 19201 rows of 16 heads of 128 (158 MB) 27 us, 5.9 TB/s (with
// four heads of a thread on their way before the angles are made 37, by ordinary stores).
template <typename T>
__global__ __launch_bounds__(kThreads) void rotate_kernel(const RotateArgs a) {
  extern __shared__ float2 angles[];
  const long long row0 = static_cast<long long>(blockIdx.x) * a.each;
  const long long left = a.turn.tokens - row0;
  const int count = left < a.each ? static_cast<int>(left) : a.each;
  make_angles(angles, a.turn, row0, 0, count);
  __syncthreads();
  const int chunks = (a.D + 15) / 16, items = count * chunks, together = kThreads / items;
  const int first = threadIdx.x / items, item = threadIdx.x - first * items;
  if (first >= together) return;
  const int t = item / chunks;
  const Chunk c = chunk_of(a.turn, item - t * chunks, a.D);
  float2 cs[8];
  if (c.turned)
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = angles[t * a.turn.pairs + (e < 4 ? c.pair0 + e : c.pair1 + e - 4)];
  const uint16_t* x = a.x + (row0 + t) * a.x_token;
  uint16_t* out = a.out + (row0 + t) * a.out_token;
  for (int h = first; h < a.heads; h += together) {
    u32x4_t u = load16(x + h * a.x_head + c.at0), v = {0, 0, 0, 0};
    if (c.at1 >= 0) v = load16(x + h * a.x_head + c.at1);
    if (c.turned) turn_chunk<T>(a.turn.adjacent, cs, u, v);
    stream16(out + h * a.out_head + c.at0, u);
    if (c.at1 >= 0) stream16(out + h * a.out_head + c.at1, v);
  }
}

// W pairs, or channels that are copied, at a time: four where sizes and alignment are multiples of
// that, or one. (19201 rows of 16 heads of 72, all of it rotated: 28 us, 3.2 TB/s; 45 one
// at a time, 40 with stores that pass the caches by, which their lines in part do not suit.)
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void rotate_any_kernel(const RotateArgs a) {
  typedef uint16_t Few __attribute__((ext_vector_type(W)));
  extern __shared__ float2 angles[];
  const long long row0 = static_cast<long long>(blockIdx.x) * a.each;
  const long long left = a.turn.tokens - row0;
  const int count = left < a.each ? static_cast<int>(left) : a.each;
  make_angles(angles, a.turn, row0, 0, count);
  __syncthreads();
  const int pairs = a.turn.pairs, turned = pairs / W, each = turned + (a.D - 2 * pairs) / W, items = count * each;
  const int side = items < kThreads ? items : kThreads, together = kThreads / side, first = threadIdx.x / side;
  if (first >= together) return;
  for (int item = threadIdx.x - first * side; item < items; item += side) {
    const int t = item / each, c = item - t * each;
    const bool turns = c < turned;
    const int at0 = turns ? (a.turn.adjacent ? 2 * W * c : W * c) : pairs + W * c;
    const int at1 = a.turn.adjacent ? at0 + W : at0 + pairs;
    float2 cs[W];
    if (turns)
#pragma unroll
      for (int e = 0; e < W; ++e) cs[e] = angles[t * pairs + W * c + e];
    const uint16_t* x = a.x + (row0 + t) * a.x_token;
    uint16_t* out = a.out + (row0 + t) * a.out_token;
#pragma unroll 2
    for (int h = first; h < a.heads; h += together) {
      Few r[2];
      r[0] = *reinterpret_cast<const Few*>(x + h * a.x_head + at0);
      if (turns) {
        r[1] = *reinterpret_cast<const Few*>(x + h * a.x_head + at1);
        auto turn = [&](float2 angle, int i, int j) {
          float x0 = T::value(r[i / W][i % W]), x1 = T::value(r[j / W][j % W]);
          turn_pair<T>(angle, x0, x1);
          const uint32_t y = T::pack(x0, x1);
          r[i / W][i % W] = static_cast<uint16_t>(y);
          r[j / W][j % W] = static_cast<uint16_t>(y >> 16);
        };
        if (a.turn.adjacent) {
#pragma unroll
          for (int e = 0; e < W; ++e) turn(cs[e], 2 * e, 2 * e + 1);
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) turn(cs[e], e, e + W);
        }
        *reinterpret_cast<Few*>(out + h * a.out_head + at1) = r[1];
      }
      *reinterpret_cast<Few*>(out + h * a.out_head + at0) = r[0];
    }
  }
}

struct RotaryAppendArgs {
  Turn turn;
  PagedView kv;
  uint16_t* ck;
  uint16_t* cv;
  float* weights;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  uint16_t* out;
  long long k_token, k_head, v_token, v_head, q_token, q_head, out_token, out_head;
  const int32_t* cu;
  int each, heads;  // each: new tokens of every sequence where cu is NULL
};

// Two workgroups per eight positions (aligned: one interleaved group of values) of a
// sequence, one for queries and keys and one for values; units are numbered as in
// paged_append_kernel. Positions before the first place count here too, since their queries
// are rotated. Bytes bound it for prompts: eight of up to 2001 tokens, 32 heads on 8 of 128
// (265 MB): 56 us, 4.7 TB/s; with ordinary loads and stores 63, 68 with all three in one workgroup,
// 72 with four heads of a thread on their way at once. A step of 32 sequences, 8 heads on 2 of 256, takes
// 5 us, latency.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void rotary_append_kernel(const RotaryAppendArgs a) {
  extern __shared__ float2 angles[];
  const bool values = blockIdx.y == 1;
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
  if (n < 1 || n > a.turn.tokens - begin || g < 0) return;  // (g < 0 where cu does not ascend)
  const int length = a.kv.length(b), first = length - n;  // position of row `begin`
  const int p0 = ((first >> 3) + g) * 8;
  if (p0 >= length) return;
  const int lo = first > p0 ? first - p0 : 0, hi = length - p0 < 8 ? length - p0 : 8;
  const long long row0 = static_cast<long long>(begin) + p0 + lo - first;  // of token lo
  const int count = hi - lo;
  const int page = p0 >= 0 ? a.kv.page(b, p0 >> a.kv.page_shift) : -1;
  const int P = 1 << a.kv.page_shift, off = p0 & (P - 1);
  if (!values) {
    // tokens x twice eight channels x heads
    constexpr int kChunks = D / 16;
    const int items = count * kChunks, together = kThreads / items;
    const int start = threadIdx.x / items, item = threadIdx.x - start * items;
    const int t = item / kChunks;
    const Chunk c = chunk_of(a.turn, item % kChunks, D);
    const int last = start < together ? a.heads + (page >= 0 ? a.kv.kv_heads : 0) : 0;
    const uint16_t* q = a.q + (row0 + t) * a.q_token;
    const uint16_t* k = a.k + (row0 + t) * a.k_token;
    uint16_t* out = a.out + (row0 + t) * a.out_token;
    make_angles(angles, a.turn, row0, p0 + lo, count);
    __syncthreads();
    float2 cs[8];
    if (c.turned && last)
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = angles[t * a.turn.pairs + (e < 4 ? c.pair0 + e : c.pair1 + e - 4)];
    uint16_t* ck = a.ck + ((static_cast<size_t>(page < 0 ? 0 : page) * a.kv.kv_heads) * P + off + lo + t) * D;
    for (int h = start; h < last; h += together) {
      const uint16_t* src = h < a.heads ? q + h * a.q_head : k + (h - a.heads) * a.k_head;
      uint16_t* dst = h < a.heads ? out + h * a.out_head : ck + static_cast<size_t>(h - a.heads) * P * D;
      u32x4_t u = load_once<u32x4_t>(src + c.at0), v = load_once<u32x4_t>(src + c.at1);
      if (c.turned) turn_chunk<T>(a.turn.adjacent, cs, u, v);
      stream16(dst + c.at0, u);
      stream16(dst + c.at1, v);
    }
    return;
  }
  if (page < 0) return;
  // values: two channels of the group's tokens, and the weights
  for (int i = threadIdx.x; i < a.kv.kv_heads * (D / 2); i += kThreads) {
    const int h = i / (D / 2), d = 2 * (i % (D / 2));
    const size_t place = (static_cast<size_t>(page) * a.kv.kv_heads + h) * P + off;
    if (a.weights && d < 16 && d / 2 >= lo && d / 2 < hi) a.weights[place + d / 2] = 0.0f;
    uint16_t* cv = a.cv + place * D;
    uint32_t pair[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= lo && e < hi)
        pair[e] = load_once<uint32_t>(a.v + (row0 + e - lo) * a.v_token + h * a.v_head + d);
    if (lo == 0 && hi == 8) {
      u32x4_t even, odd;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        even[e] = (pair[2 * e] & 0xFFFFu) | (pair[2 * e + 1] << 16);
        odd[e] = (pair[2 * e] >> 16) | (pair[2 * e + 1] & 0xFFFF0000u);
      }
      stream16(cv + 8 * d, even);
      stream16(cv + 8 * d + 8, odd);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e >= lo && e < hi) {
          cv[8 * d + e] = static_cast<uint16_t>(pair[e]);
          cv[8 * d + 8 + e] = static_cast<uint16_t>(pair[e] >> 16);
        }
    }
  }
}

// Checks a rotary plan and lays it out for the kernels.
int turn_of(const cudalm_rotary* r, const int32_t* positions, long long tokens, Turn* turn) {
  if (!r) return CUDALM_W4A16_ENULL;
  if (r->pairs < 1 || r->pairs > CUDALM_ROTARY_MAX_PAIRS || r->axes < 1 ||
      r->axes > CUDALM_ROTARY_MAX_AXES || !(r->adjacent == 0 || r->adjacent == 1) ||
      !(r->turns == 0 || r->turns == 1))
    return CUDALM_W4A16_EINVAL;
  int left[CUDALM_ROTARY_MAX_AXES] = {};
  long long sum = 0;
  for (int i = 0; i < r->axes; ++i) {
    left[i] = r->axes == 1 ? r->pairs : r->sections[i];
    if (left[i] < 0) return CUDALM_W4A16_EINVAL;
    sum += left[i];
  }
  if (sum != r->pairs) return CUDALM_W4A16_EINVAL;
  if (!r->freqs) return CUDALM_W4A16_ENULL;
  if (!aligned(r->freqs, 4) || !aligned(positions, 4)) return CUDALM_W4A16_EALIGN;
  *turn = {};
  turn->freqs = r->freqs;
  turn->positions = positions;
  turn->tokens = tokens;
  turn->pairs = r->pairs;
  turn->adjacent = r->adjacent;
  turn->scale = r->scale;
  int axis = 0;
  for (int i = 0; i < r->pairs; ++i) {
    while (left[axis] == 0) axis = (axis + 1) % r->axes;
    --left[axis];
    turn->axis[i >> 4] |= static_cast<uint32_t>(axis) << (2 * (i & 15));
    if (r->turns) axis = (axis + 1) % r->axes;
  }
  return CUDALM_W4A16_OK;
}

// Whether `n` elements can be read and written at once, n of a row on.
bool wide_rows(const cudalm_rotary_rows* q, int n) {
  return aligned(q->x, 2 * n) && aligned(q->out, 2 * n) && q->x_token_stride % n == 0 &&
         q->x_head_stride % n == 0 && q->out_token_stride % n == 0 && q->out_head_stride % n == 0;
}

// In place, an element's place has to be the same for reading and writing; and strides are no
// shorter than rows.
bool strides_fit(const cudalm_rotary_rows* q, int tokens, int D) {
  if (q->x == q->out && (q->x_token_stride != q->out_token_stride || q->x_head_stride != q->out_head_stride))
    return false;
  const int64_t t = q->out_token_stride < 0 ? -q->out_token_stride : q->out_token_stride;
  const int64_t h = q->out_head_stride < 0 ? -q->out_head_stride : q->out_head_stride;
  return (tokens < 2 || t >= D) && (q->heads < 2 || h >= D);
}

RowGrid read_rows(const cudalm_rotary_rows* q, int tokens, int D) {
  return {q->x, tokens, q->x_token_stride, q->heads, q->x_head_stride, D};
}
RowGrid written_rows(const cudalm_rotary_rows* q, int tokens, int D) {
  return {q->out, tokens, q->out_token_stride, q->heads, q->out_head_stride, D};
}

// No two rows are written to the same place, nor one where others are read.
bool written_apart(const cudalm_rotary_rows* q, int tokens, int D) {
  const RowGrid out = written_rows(q, tokens, D);
  return places_apart(out) && (q->x == q->out || !places_meet(out, read_rows(q, tokens, D)));
}

template <typename T>
int launch_append(int D, const RotaryAppendArgs& a, unsigned units, hipStream_t stream) {
  const size_t lds = sizeof(float2) * kTokens * a.turn.pairs;
  const dim3 grid(units, 2);
  if (D == 64)
    rotary_append_kernel<T, 64><<<grid, kThreads, lds, stream>>>(a);
  else if (D == 128)
    rotary_append_kernel<T, 128><<<grid, kThreads, lds, stream>>>(a);
  else
    rotary_append_kernel<T, 256><<<grid, kThreads, lds, stream>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace cudalm_hip

using namespace cudalm_hip;

extern "C" int cudalm_rotary_rotate(const cudalm_rotary* rotary, const cudalm_rotary_rows* rows,
                                    int tokens, int head_dim, int type, const int32_t* positions,
                                    hipStream_t stream) {
  RotateArgs a;
  if (const int rc = turn_of(rotary, positions, tokens, &a.turn)) return rc;
  if (!rows) return CUDALM_W4A16_ENULL;
  if (tokens < 0 || rows->heads < 0 || head_dim < 2 * rotary->pairs ||
      head_dim > 2 * CUDALM_ROTARY_MAX_PAIRS ||
      (type != CUDALM_PAGED_BF16 && type != CUDALM_PAGED_F16) || !strides_fit(rows, tokens, head_dim))
    return CUDALM_W4A16_EINVAL;
  if (tokens == 0 || rows->heads == 0) return CUDALM_W4A16_OK;
  if (!rows->x || !rows->out || !positions) return CUDALM_W4A16_ENULL;
  if (!aligned(rows->x, 2) || !aligned(rows->out, 2)) return CUDALM_W4A16_EALIGN;
  a.x = static_cast<const uint16_t*>(rows->x);
  a.out = static_cast<uint16_t*>(rows->out);
  a.x_token = rows->x_token_stride;
  a.x_head = rows->x_head_stride;
  a.out_token = rows->out_token_stride;
  a.out_head = rows->out_head_stride;
  a.heads = rows->heads;
  a.D = head_dim;
  // Fewer tokens per workgroup until the chip has some for every CU.
  a.each = kTokens;
  while (a.each > 1 && (static_cast<long long>(tokens) + a.each - 1) / a.each < 2LL * cu_count()) a.each /= 2;
  const long long groups = (static_cast<long long>(tokens) + a.each - 1) / a.each;
  if (groups >= kMaxGemmTiles) return CUDALM_W4A16_ERANGE;
  if (!written_apart(rows, tokens, head_dim)) return CUDALM_W4A16_EINVAL;
  const size_t lds = sizeof(float2) * a.each * rotary->pairs;
  auto served = [&](int n) { return wide_rows(rows, n) && rotary->pairs % n == 0 && head_dim % n == 0; };
  const bool bf16 = type == CUDALM_PAGED_BF16;
  auto kernel = served(8)   ? (bf16 ? rotate_kernel<PagedBf16> : rotate_kernel<PagedF16>)
                : served(4) ? (bf16 ? rotate_any_kernel<PagedBf16, 4> : rotate_any_kernel<PagedF16, 4>)
                            : (bf16 ? rotate_any_kernel<PagedBf16, 1> : rotate_any_kernel<PagedF16, 1>);
  kernel<<<static_cast<unsigned>(groups), kThreads, lds, stream>>>(a);
  return launch_status();
}

extern "C" int cudalm_rotary_append(const cudalm_rotary* rotary, const cudalm_paged_kv* kv,
                                    const void* k, const void* v, int64_t k_token_stride,
                                    int64_t k_head_stride, int64_t v_token_stride,
                                    int64_t v_head_stride, const cudalm_rotary_rows* queries,
                                    const int32_t* positions, const int32_t* cu_new, int tokens,
                                    hipStream_t stream) {
  if (const int rc = paged_check(kv)) return rc;
  RotaryAppendArgs a = {};
  if (const int rc = turn_of(rotary, positions, tokens, &a.turn)) return rc;
  if (tokens < 0 || (!cu_new && tokens % kv->batch) || rotary->pairs % 8 ||
      2 * rotary->pairs > kv->head_dim)
    return CUDALM_W4A16_EINVAL;
  if (queries && (queries->heads < 1 || !strides_fit(queries, tokens, kv->head_dim))) return CUDALM_W4A16_EINVAL;
  if (tokens == 0) return CUDALM_W4A16_OK;
  if (!k || !v || (queries && (!queries->x || !queries->out))) return CUDALM_W4A16_ENULL;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(cu_new, 4) || k_token_stride % 8 ||
      k_head_stride % 8 || v_token_stride % 8 || v_head_stride % 8 || (queries && !wide_rows(queries, 8)))
    return CUDALM_W4A16_EALIGN;
  const long long units = cu_new ? static_cast<long long>(tokens) / 8 + 2LL * kv->batch
                                 : static_cast<long long>(kv->batch) * (tokens / kv->batch / 8 + 2);
  if (units >= kMaxGemmTiles / 2 || kv->kv_heads >= (1 << 22) || (queries && queries->heads >= (1 << 22)))
    return CUDALM_W4A16_ERANGE;
  if (queries) {
    const RowGrid out = written_rows(queries, tokens, kv->head_dim);
    if (!written_apart(queries, tokens, kv->head_dim) ||
        places_meet(out, {k, tokens, k_token_stride, kv->kv_heads, k_head_stride, kv->head_dim}) ||
        places_meet(out, {v, tokens, v_token_stride, kv->kv_heads, v_head_stride, kv->head_dim}))
      return CUDALM_W4A16_EINVAL;
  }
  a.kv = view_of(kv);
  a.ck = static_cast<uint16_t*>(kv->k);
  a.cv = static_cast<uint16_t*>(kv->v);
  a.weights = kv->weights;
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  if (queries) {
    a.q = static_cast<const uint16_t*>(queries->x);
    a.out = static_cast<uint16_t*>(queries->out);
    a.q_token = queries->x_token_stride;
    a.q_head = queries->x_head_stride;
    a.out_token = queries->out_token_stride;
    a.out_head = queries->out_head_stride;
    a.heads = queries->heads;
  }
  a.cu = cu_new;
  a.each = cu_new ? 0 : tokens / kv->batch;
  return kv->type == CUDALM_PAGED_BF16
             ? launch_append<PagedBf16>(kv->head_dim, a, static_cast<unsigned>(units), stream)
             : launch_append<PagedF16>(kv->head_dim, a, static_cast<unsigned>(units), stream);
}
