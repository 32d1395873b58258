// Device vocabulary of the paged cache in 8 bits (kv_append_normed, kv8_read, kv8_attention): codes, their blocks and
// scales. Private to csrc/kernels.
#pragma once

#include "paged_common.h"

namespace gie_hip {

constexpr int kKvBlock = 16;  // positions of a head that share a scale
// No block counts as smaller than this: a scale of 0 would have no reciprocal, and the attention divides sums by a
// block's scale, which stays far inside FP32's range so.
constexpr float kKvLeast = 0x1p-64f;

// Codes: divide gives x / scale, correctly rounded to FP32: the product with the correctly rounded reciprocal and one
// correction by its residual (Markstein's division; without the correction a quotient is off by a step now and then,
// and values that lie halfway between two codes are common: half of a block's largest is 63.5). It costs two instructions
// a value and hardly any time (int8, 4 prompts of 8192 tokens with 32 + 2 * 8 heads of 128, appended and read back: 200.4 us,
// 199.7 without).
// encode4 rounds four quotients to nearest even, byte by byte; they are within the largest code but for FP32's rounding,
// which does not reach the next step. decode4 gives bytes 0 and 2, and 1 and 3, as FP16 times 1 / kUnit, exactly (five
// instructions in both types; bytes 0 and 1 together would take one or two more).
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
struct Int8Code {
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ float scale(float most) { return fmaxf(most, kKvLeast) / 127.f; }
  static __device__ __forceinline__ float divide(float x, float scale, float inv) {  // inv: 1 / scale, rounded
    const float q = x * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, scale, x), inv, q);
  }
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    // added to 1.5 2^23 a value is rounded to a whole number in the lowest bits
    const auto whole = [](float x) { return __float_as_uint(x + 12582912.f); };
    const uint32_t lo = __builtin_amdgcn_perm(whole(b), whole(a), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(whole(d), whole(c), 0x04000c0cu);
    return lo | hi;
  }
  static __device__ __forceinline__ float decode1(uint32_t code) { return float(int8_t(code)); }
  static __device__ __forceinline__ u32x2 decode4(uint32_t w) {
    // code + 128 as the low bits of 1024, less 1152
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t even = __builtin_amdgcn_perm(0x64646464u, x, 0x04020400u);
    const uint32_t odd = __builtin_amdgcn_perm(0x64646464u, x, 0x04030401u);
    const f16x2 less = {_Float16(-1152.f), _Float16(-1152.f)};
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, even) + less),
                 __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, odd) + less)};
  }
};

// e4m3 with a power of 2 as scale: a larger scale moves exponents alone, so codes that are rounded again keep their bits
// unless they fall among the subnormals.
struct E4m3Code {
  static constexpr float kUnit = 256.f;  // bits moved into FP16's fields stand for 2^(7 - 15) of the value
  static __device__ __forceinline__ float scale(float most) {
    const uint32_t bits = __float_as_uint(fmaxf(most, kKvLeast));  // 448 = 1.75 2^8
    return __uint_as_float(((bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u)) << 23);
  }
  static __device__ __forceinline__ float divide(float x, float scale, float inv) { return x * inv; }  // a power of 2
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
  }
  static __device__ __forceinline__ float decode1(uint32_t code) {  // the NaN codes (0x7f, 0xff) become 480
    return float(__builtin_bit_cast(_Float16, uint16_t((code & 0x80u) << 8 | (code & 0x7fu) << 7))) * kUnit;
  }
  static __device__ __forceinline__ u32x2 decode4(uint32_t w) {
    // a code in the upper byte, moved down by one with its sign kept: the sign's copy and what the lower byte left go
    const auto down = [](uint32_t x) {
      const s16x2 y = __builtin_bit_cast(s16x2, x) >> s16x2{1, 1};
      return __builtin_bit_cast(uint32_t, y) & 0xbf80bf80u;
    };
    return u32x2{down(w << 8), down(w)};
  }
};

// The block of a slot of a sequence's new tokens: positions [first, end) are new, the block's own start at `start`;
// none: first >= end. page -1: not stored.
struct Block {
  int start, first, end, page, slot;
  int row0;  // row of q, k, v of position `first`
};
__device__ __forceinline__ Block block_of(const gie_kv_geom& g, const int* __restrict__ q_starts,
                                          const int* __restrict__ seq_lens, const int* __restrict__ page_table, int slot) {
  // n tokens from any position on touch at most n / 16 + 2 blocks, so sequence b's slots start at floor(first / 16) + 2 b
  const auto from = [&](int first, int b) { return min(max(first, 0), g.total_tokens) / kKvBlock + 2 * b; };
  const Sequence s = locate(q_starts, seq_lens, g.batch, g.total_tokens, slot, from);
  const int p0 = max(s.base, 0), at = slot - from(s.first, s.index);
  const int p1 = int(min((long long)s.base + s.count, (long long)g.max_pages * g.page_size));
  Block r;
  r.start = (p0 / kKvBlock + at) * kKvBlock;
  r.first = max(r.start, p0);
  r.end = at >= 0 ? min(r.start + kKvBlock, p1) : r.first;
  r.row0 = s.first + (r.first - s.base);
  r.page = -1;
  r.slot = 0;
  if (r.first < r.end) {
    const int row = r.start / g.page_size;
    const int page = page_table[(long long)s.index * g.max_pages + row];
    if (page >= 0 && page < g.num_pages) r.page = page;
    r.slot = r.start - row * g.page_size;
  }
  return r;
}
inline long long block_slots(const gie_kv_geom& g) { return (long long)g.total_tokens / kKvBlock + 2ll * g.batch; }

inline bool valid_code(int code) { return code == GIE_HIP_KV_INT8 || code == GIE_HIP_KV_E4M3; }

}  // namespace gie_hip
