// What the paged key-value kernels share (gfx950): element types, values that are
// not finite, the pages of a tile, which tokens a query sees.
#ifndef CUDALM_PAGED_DEVICE_H
#define CUDALM_PAGED_DEVICE_H

#include "cudalm_paged_kv.h"
#include "hip_common.h"

namespace cudalm_hip {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// 16-bit element types: matrix products with fp32 accumulation, and rounding
// (to nearest even) of pairs.
struct PagedBf16 {
  static constexpr uint32_t kExp = 0x7F80u;  // an all-ones exponent: Inf or NaN
  static constexpr uint32_t kExpLow = 0x0080u, kOne = 0x3F80u;
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return mfma16(a, b, c);
  }
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return f32_to_bf16_rne2(lo, hi);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return bf16_lo(x); }
};

struct PagedF16 {
  static constexpr uint32_t kExp = 0x7C00u;
  static constexpr uint32_t kExpLow = 0x0400u, kOne = 0x3C00u;
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
  }
  static __device__ __forceinline__ float value(uint16_t x) {
    return static_cast<float>(__builtin_bit_cast(_Float16, x));
  }
};

// Running maxima start here and not at -inf, so that differences of maxima
// are never inf - inf; no finite score is below it.
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f;

// A hidden token's weight of zero times a value of Inf or NaN is NaN in a matrix
// product. Where some row sees only part of a tile and its values are not all
// finite, the product takes them without those (finite_part), and the rows that
// do see them get theirs from two more products of whole numbers: how many
// tokens that a row sees (ones in `seen_operand`) hold +Inf or NaN, and how
// many -Inf or NaN (special_part). The one gives Inf, the other -Inf, whatever the
// tokens' weights: also where they underflow, in a part or in the join of parts, so
// that results do not depend on how a call is cut.
// Both halves of a word at once: an all-ones exponent plus its lowest bit carries
// into bit 15, a mantissa that is not zero plus its mask into the exponent.
template <typename T>
__device__ __forceinline__ uint32_t special_bits(uint32_t v) {
  return ((v & T::kExp * 0x10001u) + T::kExpLow * 0x10001u) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t special_bits(u32x4_t v) {
  return special_bits<T>(v[0]) | special_bits<T>(v[1]) | special_bits<T>(v[2]) | special_bits<T>(v[3]);
}
template <typename T>
__device__ __forceinline__ u32x4_t finite_part(u32x4_t v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] &= ~((special_bits<T>(v[i]) >> 15) * 0xFFFFu);
  return v;
}
// Ones where v is Inf of the sign that `flip` (0: negative, all ones: positive)
// leaves set in bit 15, or NaN.
template <typename T>
__device__ __forceinline__ u32x4_t special_part(u32x4_t v, uint32_t flip) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t low = T::kExpLow * 0x10001u, mantissa = low - 0x10001u;
    const uint32_t nan = ((v[i] & mantissa) + mantissa) & low;
    v[i] = ((special_bits<T>(v[i]) & ((v[i] ^ flip) | nan * (0x8000u / T::kExpLow))) >> 15) * T::kOne;
  }
  return v;
}
// Ones for the eight tokens of the low bits of `seen`.
template <typename T>
__device__ __forceinline__ u32x4_t seen_operand(uint32_t seen) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = ((seen >> (2 * i)) & 1 ? T::kOne : 0u) | ((seen >> (2 * i + 1)) & 1 ? T::kOne << 16 : 0u);
  return r;
}

// The larger of a lane's x and that of the lane 32 (16) away: one exchange of half
// waves (of odd rows of 16 lanes with even ones) in the vector unit, where a
// shuffle goes through the LDS.
__device__ __forceinline__ float max_across_32(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float max_across_16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A load that no store of the kernel changes, from a wave-uniform address.
__device__ __forceinline__ int load_uniform(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(p));
}

// Lane x's 64-bit value. (The builtin's result is signed: without the casts a low word
// from 2^31 on would fill the high one.)
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int x) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v), x));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), x));
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// The cache as the kernels take it.
struct PagedView {
  const int32_t* tables;
  const int32_t* lens;
  int num_pages, page_shift, kv_heads, batch, max_pages;

  __device__ __forceinline__ int length(int b) const {
    const int n = lens[b], cap = max_pages << page_shift;
    return n < 0 ? 0 : n < cap ? n : cap;
  }
  // length() for a wave-uniform argument: a scalar load.
  __device__ __forceinline__ int uniform_length(int b) const {
    const int n = load_uniform(lens + b), cap = max_pages << page_shift;
    return n < 0 ? 0 : n < cap ? n : cap;
  }
  // The page of table entry i of sequence b; -1 where these tokens are absent.
  __device__ __forceinline__ int page(int b, int i) const {
    if (i >= max_pages) return -1;
    const int p = tables[static_cast<size_t>(b) * max_pages + i];
    return p >= 0 && p < num_pages ? p : -1;
  }
};

// Tiles of 2^tile_shift tokens that some query of positions first .. last
// sees: the tiles of the sinks, then those from the earliest window's first
// token on.
struct PagedTiles {
  int sink_tiles, from, count;

  __device__ __forceinline__ PagedTiles(int length, int first, int last, int window, int sinks,
                                        int tile_shift) {
    const int mask = (1 << tile_shift) - 1;
    sink_tiles = 0;
    from = 0;
    if (window > 0 && first - window + 1 > 0) {
      const int s = sinks < length ? sinks : length;
      const int st = (s + mask) >> tile_shift, w = (first - window + 1) >> tile_shift;
      if (w > st) sink_tiles = st, from = w - st;
    }
    const int end = (last + 1 + mask) >> tile_shift;
    count = end - from > 0 ? end - from : 0;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : i + from; }
};

__device__ __forceinline__ bool paged_sees(int t, int p, int window, int sinks) {
  return t <= p && (window <= 0 || t > p - window || t < sinks);
}

// A part's sum under the weight that the join gives it: Inf and NaN of values that a
// row sees stay, also under a weight that has underflowed.
__device__ __forceinline__ float joined(float w, float sum) {
  return w == 0.0f && !(fabsf(sum) < __builtin_inff()) ? sum : w * sum;
}

// How many of `tiles` tiles each of at most `splits` parts takes: the least the
// host asks for, more where that would leave tiles over.
__device__ __forceinline__ int tiles_per_split(int tiles, int splits, int least) {
  const int c = (tiles + splits - 1) / splits;
  return c > least ? c : least;
}

// The sequence whose units contain unit u, where sequence b's begin at
// cu[b] * mul / per + extra * b: 64 sequences per step, a ballot each. -1: none.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int u, int mul, int per,
                                           int extra) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int b = b0 + lane;
    const int n = __popcll(__ballot(b < batch && cu[b] * mul / per + extra * b <= u));
    count += n;
    if (n < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(count) - 1;
}

inline int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

inline PagedView view_of(const cudalm_paged_kv* kv) {
  return {kv->tables,   kv->lens,  kv->num_pages, log2_of(kv->page_size),
          kv->kv_heads, kv->batch, kv->max_pages};
}

// Argument checks that all entry points share (paged_cache.hip).
int paged_check(const cudalm_paged_kv* kv);
int paged_check_query(const cudalm_paged_kv* kv, const cudalm_paged_query* q);

// Cached tokens a sequence is expected to have at most.
inline int expected_len(const cudalm_paged_kv* kv, int max_len) {
  const int cap = kv->max_pages * kv->page_size;
  return max_len > 0 && max_len < cap ? max_len : cap;
}

// A window that hides nothing is none; positions fit 30 bits.
inline int window_of(const cudalm_paged_query* q) {
  return q->window <= 0 || q->window >= (1 << 30) ? 0 : q->window;
}
inline int sinks_of(const cudalm_paged_query* q) {
  return q->sinks <= 0 ? 0 : q->sinks < (1 << 30) ? q->sinks : 1 << 30;
}

}  // namespace cudalm_hip

#endif
