// What the attention kernels over a paged cache (paged_attention, kv8_attention) share: their arguments, tiles of rows and
// ranges of keys, capped scores, the join of parts and the choice of a launch shape. Private to csrc/kernels.
#pragma once

#include <cmath>

#include "paged_common.h"

#include "lds_pipe.h"

namespace gie_hip {

typedef __attribute__((address_space(4))) const int const_int;  // uniform loads through the scalar cache
typedef __attribute__((address_space(3))) u32x4 lds_v4;
typedef __attribute__((address_space(3))) u32x2 lds_v2;
typedef __attribute__((address_space(3))) int lds_i;
typedef __attribute__((address_space(3))) long long lds_ll;
typedef __attribute__((address_space(3))) f32x4 lds_f4;
typedef short v4s __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const uint16_t* q;
  const int* q_starts;
  const int* seq_lens;
  const int* page_table;
  uint16_t* out;
  float* part;  // splits > 1: [row = token * q_heads + head][split][head_dim + 4]: O, m (in powers of 2), l, two unused
  long long q_stride, o_stride;
  int batch, total_tokens, q_heads, kv_heads, group;
  int page16, num_pages, max_pages;  // page16: a page's size in units of 16 positions
  unsigned page_magic;               // division by page16
  int page_shift;
  int capacity;  // max_pages * page_size
  int window, sinks;  // sinks: 0 without a window
  float mult;      // a score's power of 2: the product times this, or (cap > 0) what the cap leaves of it times this
  float cap_in, cap;  // cap > 0: cap * tanh(product * cap_in / (2 log2(e)))
  int negate;      // a negative scale: q changes its sign, so that the largest product is the largest score
  int splits, chunk;  // parts of the keys and the fewest tiles of one
};

template <int D>
constexpr int kPitch = D == 96 ? 256 : 2 * D;  // bytes of a row in LDS

// permutation of a row's 16-byte chunks: of keys, read as 16 bytes of 16 rows at a time, and of values, read as 64
// bytes of 4 rows at a time
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  return (D == 64 ? (row >> 1) & 1 : row & 3) << 2;
}

__device__ __forceinline__ int div_magic(int n, unsigned magic, int shift) {
  return int((__umulhi(unsigned(n), magic) + unsigned(n)) >> shift);
}

__device__ __forceinline__ float swap_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_add(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a 16-lane group reads 4 rows of 16 values; each lane gets the 4 rows' values of its column
__device__ __forceinline__ u32x2 read_transposed(unsigned at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       reinterpret_cast<__attribute__((address_space(3))) v4s*>(size_t(at))));
}

// bits 15 and 31: whether the lower and the upper half hold an infinity or a NaN (the exponent's ones carry over)
template <typename E>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  constexpr uint32_t mask = E::kDtype == GIE_HIP_FP16 ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = E::kDtype == GIE_HIP_FP16 ? 0x04000400u : 0x00800080u;
  return ((x & mask) + one) & 0x80008000u;
}

// Scores under a cap. 1 - 2 / (2^z + 1) is off by about 2^-23 however small z is, and the score by the cap times that:
// less than what the sum of a product is off by, up to caps of kExpCap.
constexpr float kTwoLog2E = 2.f * 1.44269504088896341f, kExpCap = 64.f;
__device__ __forceinline__ void cap_scores(const AttnArgs& a, f32x16& s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float e = __builtin_amdgcn_exp2f(s[i] * a.cap_in);
    s[i] = a.cap - 2.f * a.cap * __builtin_amdgcn_rcpf(e + 1.f);
  }
}
// Under a cap past kExpCap, in units of the product x = s[i]: where |x / cap| < 0.2 the odd polynomial of tanh, times x
// itself (its next term is 2^-30 of it), so that scores keep FP32's relative precision under any cap; the exponential
// only where a wave has a larger one. In a kernel of its own: beside the other form it took 1 % from calls that need
// neither (registers, a longer loop). Two prompts of 4096 tokens, 32 heads of 128, scores around 1: 362 us under a cap of
// 65, 352 under one of 50.
__device__ __forceinline__ void cap_products(const AttnArgs& a, f32x16& s) {
  constexpr float kBound = 0.2f * kTwoLog2E, k2 = 1.f / (kTwoLog2E * kTwoLog2E);
  const auto polynomial = [](float x, float z) {
    const float z2 = z * z;
    float p = __builtin_fmaf(z2, 62.f / 2835.f * k2 * k2 * k2 * k2, -17.f / 315.f * k2 * k2 * k2);
    p = __builtin_fmaf(z2, p, 2.f / 15.f * k2 * k2);
    p = __builtin_fmaf(z2, p, -1.f / 3.f * k2);
    return x * __builtin_fmaf(z2, p, 1.f);
  };
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(s[i]));
  if (!__any(most * a.cap_in >= kBound)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = polynomial(s[i], s[i] * a.cap_in);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float z = fabsf(s[i] * a.cap_in), r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.f);
      const float t = __builtin_copysignf(a.cap * __builtin_fmaf(-2.f, r, 1.f), s[i]);
      s[i] = z < kBound ? polynomial(s[i], z) : t;  // a NaN stays one
    }
  }
}

// the part of a sequence's keys that a tile of rows reads, in tiles of TT positions, and its division: sink_tiles tiles
// from position 0 on, which end before lo, then tiles over [lo, hi), lo a multiple of 16
struct KeyRange {
  int lo, hi, sink_tiles;
  int tiles;      // all of them
  int per_split;  // tiles
  int splits;     // parts that hold any
};
template <int TT>
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, int pos_first, int pos_last) {
  KeyRange r;
  r.hi = min(pos_last + 1, a.capacity);
  r.lo = a.window > 0 ? max(0, pos_first - a.window + 1) & ~15 : 0;
  r.lo = min(r.lo, max(r.hi, 0) & ~15);
  r.sink_tiles = (a.sinks + TT - 1) / TT;
  if (r.sink_tiles * TT >= r.lo) r.lo = r.sink_tiles = 0;  // they meet the window
  r.tiles = r.sink_tiles + (r.hi > r.lo ? (r.hi - r.lo + TT - 1) / TT : 0);
  r.per_split = max(a.chunk, (r.tiles + a.splits - 1) / a.splits);
  r.splits = (r.tiles + r.per_split - 1) / r.per_split;
  return r;
}

// a position that a row at `pos` sees (oldest: pos - window, or -1 without one)
__device__ __forceinline__ bool sees(const AttnArgs& a, int key, int pos, int oldest) {
  return key <= pos && (key > oldest || key < a.sinks);
}

// rows of a tile: its sequence, the first of its rows; position(r) = seq.base + r / group
struct RowTile {
  Sequence seq;
  int row0, rows;  // rows: valid ones from row0 on, <= 0: none
};
template <int R>
__device__ __forceinline__ RowTile row_tile(const AttnArgs& a, int slot) {
  // sequence b's tiles start at slot floor(q_starts[b] * group / R) + b: as many slots as it can need lie before the next
  // one's, whatever it holds
  const auto start = [&](int first, int b) {
    return int((long long)min(max(first, 0), a.total_tokens) * a.group / R) + b;
  };
  RowTile t;
  t.seq = locate(a.q_starts, a.seq_lens, a.batch, a.total_tokens, slot, start);
  t.row0 = (slot - start(t.seq.first, t.seq.index)) * R;
  t.rows = t.row0 >= 0 ? t.seq.count * a.group - t.row0 : 0;
  return t;
}

// Joins the parts of the keys: WAVES waves for each row (token, head), lanes over the head's values 4 at a time, the parts
// dealt out to the groups of lanes that this leaves. One wave (4 rows to a workgroup) where there are few parts and many
// rows, four where one row has dozens of parts.
namespace {
template <typename E, int D, int R, int TT, int WAVES>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  constexpr int kLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, kInWave = 64 / kLanes, kGroups = WAVES * kInWave;
  __shared__ f32x4 sums[WAVES][kLanes];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = WAVES > 1 ? tid >> 6 : 0;
  const long long row = WAVES > 1 ? blockIdx.x : blockIdx.x * 4ll + (tid >> 6);
  if (row >= (long long)a.total_tokens * a.q_heads) return;
  const int token = int(row / a.q_heads), head = int(row % a.q_heads);
  const float* part = a.part + row * a.splits * (D + 4);
  const Sequence seq =
      locate(a.q_starts, a.seq_lens, a.batch, a.total_tokens, token, [](int first, int) { return first; });
  if (token < seq.first || token >= seq.first + seq.count) return;
  const int row0 = ((token - seq.first) * a.group + head % a.group) / R * R;
  const int last_row = min(row0 + R, seq.count * a.group) - 1;
  const int splits = key_range<TT>(a, seq.base + row0 / a.group, seq.base + last_row / a.group).splits;
  if (splits <= 1) return;  // written already
  float top = -INFINITY;
  for (int z = lane; z < splits; z += 64) top = fmaxf(top, part[z * (D + 4) + D]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top;
  // a part without a maximum weighs 1: it holds zeros, or a NaN that has to stay
  const auto weight = [&](float m) { return m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref); };
  float total = 0.f;
  for (int z = lane; z < splits; z += 64) total += part[z * (D + 4) + D + 1] * weight(part[z * (D + 4) + D]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
  const int at = lane % kLanes, group = wave * kInWave + lane / kLanes;
  f32x4 v = {};
  if (at * 4 < D) {
#pragma unroll 4
    for (int z = group; z < splits; z += kGroups)
      v += *reinterpret_cast<const f32x4*>(part + z * (D + 4) + at * 4) * weight(part[z * (D + 4) + D]);
  }
#pragma unroll
  for (int d = kLanes; d < 64; d <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], d);
  if (WAVES > 1) {
    if (lane < kLanes) sums[wave][at] = v;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += sums[w][at];
  }
  if (lane >= kLanes || at * 4 >= D) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  uint16_t* dst = a.out + token * a.o_stride + head * D + at * 4;
  if (total == 0.f) v = f32x4{};
  v *= inv;
  store_8_bytes(dst, u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])});
}

}  // namespace

// ---- launch shape: the same on both sides of the workspace query ----
struct Shape {
  bool wide;  // rows of a workgroup: 128 that share tiles of 64 keys, or 32 with tiles of 32 for each wave
  int slots, splits, chunk;
};

constexpr int kNarrowRows = 32, kWideRows = 128, kNarrowKeys = 32, kWideKeys = 64;  // a tile's

inline Shape shape_of(const gie_kv_geom& g) {
  Shape s;
  const int group = g.q_heads / g.kv_heads;
  const long long rows = (long long)g.total_tokens * group;
  const int most_new = g.max_new > 0 ? g.max_new : (g.total_tokens + g.batch - 1) / g.batch;
  s.wide = (long long)most_new * group > kNarrowRows;
  const int R = s.wide ? kWideRows : kNarrowRows, tt = s.wide ? kWideKeys : kNarrowKeys;
  s.slots = int(rows / R) + g.batch;
  // tiles of rows that hold any, about
  const long long busy = (rows + R - 1) / R > g.batch ? (rows + R - 1) / R : g.batch;
  long long len = (long long)g.max_pages * g.page_size;
  if (g.max_len > 0 && g.max_len < len) len = g.max_len;
  if (g.window > 0 && (long long)g.window + most_new + g.sinks < len) len = (long long)g.window + most_new + g.sinks;
  const long long tiles = (len + tt - 1) / tt;
  const long long blocks = busy * g.kv_heads;
  const int fewest = s.wide ? 2 : 8;  // tiles of a part
  const long long most = tiles / fewest > 1 ? tiles / fewest : 1;
  long long splits = 1;
  if (!s.wide) {
    // Bytes bound: one workgroup for each compute unit, whose LDS holds 64 KiB and more on their way; over 8 bits at
    // head_dim 64 it is half of that and a second workgroup would fit, which this rule does not use (one token over 65536,
    // 8 key heads: 20.6 us with the join's launch, 14.2 of bytes).
    splits = 256 / blocks;
  } else {
    // Products: what a tile of 64 keys takes on a compute unit by itself, and the share of one that two workgroups have,
    // us as measured (head_dim 64, 96, 128: 1.5, 1.8, 2.0 by itself over caches of their own, 1.4 at 128 over a shared
    // one, 1.08 shared; capped scores 0.75 more; head_dim 256, where one fits: 3.5). The device's share of all tiles, and
    // as much of a part's path as the parts differ in length (a prompt's rows see from nothing to all of it). Parts: a
    // launch, and their sums written and read once. Measured / so estimated, us: 512 tokens over 7680 in 4 parts 93 / 88,
    // in 2 113 / 112; one prompt of 4096, 16 heads, whole 118 / 138, in 2 parts 178 / 131 (so only 10 % less counts).
    const bool single = g.head_dim == 256;
    const double size = g.head_dim / 128.0, cap = g.softcap > 0 ? 0.7 : 0;
    const double alone = single ? 3.5 : 0.9 + 0.6 * size + cap, shared = single ? 3.5 : 0.5 + 0.58 * size + cap;
    const double mean = tiles - (most_new < len ? most_new : len) / (2.0 * tt), uneven = 1 - mean / tiles;
    double best = 0;
    for (long long n = 1; n <= most && n <= 64; ++n) {
      const long long each = (blocks * n + 255) / 256;  // workgroups of a compute unit
      const double path = (each == 1 || single ? alone : 2 * shared) * double((tiles + n - 1) / n);
      const double share = shared * blocks * mean / 256 + uneven * path;
      const double join = n == 1 ? 0 : 4 + 2.0 * rows * g.kv_heads * n * (g.head_dim + 4) * 4 / 5e6;
      const double us = (path > share ? path : share) + join;
      if (n == 1 || us < 0.9 * best) best = us, splits = n;
    }
  }
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  s.chunk = int((tiles + splits - 1) / splits);
  s.splits = int((tiles + s.chunk - 1) / s.chunk);
  return s;
}

template <typename K, typename A>
int start(K kernel, int grid, int threads, int lds_bytes, hipStream_t stream, const A& a) {
  const int rc = set_lds_limit(reinterpret_cast<const void*>(kernel), lds_bytes);
  if (rc != GIE_HIP_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(unsigned(threads)), unsigned(lds_bytes), stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

// joins what a launch left in parts
template <typename E, int D>
int join_parts(const AttnArgs& a, const Shape& s, hipStream_t stream) {
  const long long rows = (long long)a.total_tokens * a.q_heads;
  const bool many = s.splits > 8;
  const auto join =
      s.wide ? (many ? join_kernel<E, D, kWideRows, kWideKeys, 4> : join_kernel<E, D, kWideRows, kWideKeys, 1>)
             : (many ? join_kernel<E, D, kNarrowRows, kNarrowKeys, 4> : join_kernel<E, D, kNarrowRows, kNarrowKeys, 1>);
  hipLaunchKernelGGL(join, dim3(unsigned(many ? rows : (rows + 3) / 4)), dim3(256), 0, stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
// whether a launch and its join have as many threads as the device takes
inline bool fits_launch(const AttnArgs& a, const Shape& s) {
  const long long grid = (long long)s.slots * s.splits * a.kv_heads;
  const long long rows = (long long)a.total_tokens * a.q_heads;
  const long long joining = s.splits == 1 ? 0 : s.splits > 8 ? rows * 256 : rows * 64;
  return grid * 512 <= 0xffffffffll && joining <= 0xffffff00ll;
}

inline size_t parts_bytes(const gie_kv_geom& g, const Shape& s) {
  return s.splits == 1 ? 0 : size_t(g.total_tokens) * g.q_heads * s.splits * (g.head_dim + 4) * sizeof(float);
}

inline bool valid_attention(const gie_kv_geom* g, const void* q, const void* k_pages, const void* v_pages,
                            const int* q_starts, const int* seq_lens, const int* page_table, const void* out) {
  if (!q || !k_pages || !v_pages || !q_starts || !seq_lens || !page_table || !out || q == out) return false;
  return aligned_to(q, 2) && aligned_to(out, 2) && aligned_to(k_pages, 16) && aligned_to(v_pages, 16);
}

// the arguments but for the cache's pages; returns whether the cap is past kExpCap
inline bool fill_args(AttnArgs& a, const gie_kv_geom* g, const Shape& shape, const void* q, const int* q_starts,
                      const int* seq_lens, const int* page_table, void* out, void* workspace) {
  a.q = static_cast<const uint16_t*>(q);
  a.q_starts = q_starts;
  a.seq_lens = seq_lens;
  a.page_table = page_table;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  a.q_stride = g->q_stride;
  a.o_stride = g->o_stride;
  a.batch = g->batch;
  a.total_tokens = g->total_tokens;
  a.q_heads = g->q_heads;
  a.kv_heads = g->kv_heads;
  a.group = g->q_heads / g->kv_heads;
  a.page16 = g->page_size / 16;
  a.num_pages = g->num_pages;
  a.max_pages = g->max_pages;
  // n / page16 = (umulhi(n, magic) + n) >> shift for n < 2^31: shift = ceil(log2(page16)), magic = 2^32 (2^shift /
  // page16 - 1), rounded up
  int shift = 0;
  while ((1ll << shift) < a.page16) ++shift;
  a.page_shift = shift;
  a.page_magic = unsigned(((((1ull << shift) - unsigned(a.page16)) << 32) / unsigned(a.page16)) + 1);
  a.capacity = g->max_pages * g->page_size;
  a.window = g->window < a.capacity ? g->window : 0;  // no position lies further back
  a.sinks = a.window == 0 ? 0 : g->sinks < a.capacity ? g->sinks : a.capacity;
  constexpr float kLog2E = 1.44269504088896341f;
  const float scale = g->scale < 0 ? -g->scale : g->scale;
  a.negate = g->scale < 0;
  // factors stay finite, or a product of 0 would become a NaN
  a.mult = fminf(scale * kLog2E, 3e38f);
  bool large_cap = false;
  if (g->softcap > 0) {
    a.cap_in = fminf(kTwoLog2E * (scale / g->softcap), 3e38f);
    large_cap = g->softcap > kExpCap;
    if (!large_cap) {
      a.mult = kLog2E;
      a.cap = g->softcap;
    } else {
      a.cap = fminf(g->softcap / scale, 3e38f);
    }
  }
  a.splits = shape.splits;
  a.chunk = shape.chunk;
  return large_cap;
}

}  // namespace gie_hip
