// Attention of new tokens over a paged key/value cache:
//   out[t][h] = sum_j softmax_j(s_j) v_j,  s_j = scale * q[t][h] . k_j  (or softcap * tanh(that / softcap)),
// over the positions j <= p (and j > p - window) of the token's sequence, in one pass over the keys with the running
// maximum m and sum l of the softmax.
//
// Rows. All (token, head) pairs of a sequence that read one key head are rows of one matrix, r = token * group + head in
// group, so a tile of rows shares every key it reads and one token of a grouped head fills part of a tile instead of a
// row of it. A workgroup takes WR * 32 rows of one key head of one sequence, and the z-th part of their keys.
//
// Products. Both are 32x32x16 MFMAs with the rows in the columns: S^T = K Q^T leaves a lane 16 scores (keys) of one row
// for each 32 keys, so maxima and sums are a lane's own but for one exchange between the wave's halves, and the rescaling
// of O^T = V^T P^T is a product by a lane's own number. The order of the summed keys in the second product is free: it
// takes keys {4h..4h+3, 8+4h..8+4h+3} of 16 from half h, which is how S^T left them, so P never leaves its registers;
// V comes out of LDS in that order with ds_read_b64_tr_b16.
//
// Keys and values travel HBM -> LDS by direct loads, 16 positions at a time (a page holds a multiple of 16, so they are
// contiguous), through a buffer resource that ends at the last position anyone sees: what lies behind it, or in a page
// outside the cache, arrives as zeros. 16-byte chunks of a row are permuted by the row so that the fragment reads meet
// no bank twice in a phase. The waves of a workgroup either share a tile of keys (WR > 1: one barrier for each tile) or
// take tiles of their own (WR == 1, WK waves, no barrier until their results are joined).
//
// Few rows (one token of a grouped head: up to 32) are bound by the cache's bytes: one token over 32768 positions of 8
// key heads of 128 in 32 parts 24 us + 4 for the join, 4.6 TB/s in all; a step of 64 sequences 219 us, 5.0 TB/s (a large
// copy reaches 4.7). Many rows are bound by the products: two prompts of 4096 tokens, 32 heads of 128, 288-311 us, 0.88 to
// 0.95 PFLOP/s (a large library product 1.23); 2048 tokens over 30000 1.0. Matrix cores are busy 0.42 of the time, the
// vector unit (softmax) 0.47 and LDS 0.35, on two workgroups of 4 waves for each compute unit (BF16): measured (at 310 us
// for a call, before q and out went through LDS) without exponentials -5 %, without any softmax -13 %, without loads
// -16 %. At that time 64 rows for each wave (half the LDS reads, one wave for each SIMD) took 408 us, eight waves sharing
// a tile 318 and more for ragged batches.
// The weights enter the second product in the storage type, since the matrix cores take FP32 at a sixteenth of the rate:
// outputs are off by 2.1e-3 to 2.3e-3 of their size in BF16 and 2.8e-4 in FP16, where the same in FP32 with one rounding
// at the end has 1.7e-3 and 2.1e-4.
#include <cmath>

#include "paged_common.h"

#include "lds_pipe.h"

namespace gie_hip {
namespace {

typedef __attribute__((address_space(4))) const int const_int;  // uniform loads through the scalar cache
typedef __attribute__((address_space(3))) u32x4 lds_v4;
typedef __attribute__((address_space(3))) u32x2 lds_v2;
typedef __attribute__((address_space(3))) int lds_i;
typedef __attribute__((address_space(3))) long long lds_ll;
typedef __attribute__((address_space(3))) f32x4 lds_f4;
typedef short v4s __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const uint16_t* q;
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  const int* q_starts;
  const int* seq_lens;
  const int* page_table;
  uint16_t* out;
  float* part;  // splits > 1: [row = token * q_heads + head][split][head_dim + 2]: O, m (in powers of 2), l
  long long q_stride, o_stride;
  int batch, total_tokens, q_heads, kv_heads, group;
  int page16, num_pages, max_pages;  // page16: a page's size in units of 16 positions
  unsigned page_magic;               // division by page16
  int page_shift;
  int capacity;  // max_pages * page_size
  int window;
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

// the part of a sequence's keys that a tile of rows reads, in tiles of TT positions, and its division
struct KeyRange {
  int lo, hi;     // positions [lo, hi), lo a multiple of 16
  int per_split;  // tiles
  int splits;     // parts that hold any
};
template <int TT>
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, int pos_first, int pos_last) {
  KeyRange r;
  r.hi = min(pos_last + 1, a.capacity);
  r.lo = a.window > 0 ? max(0, pos_first - a.window + 1) & ~15 : 0;
  r.lo = min(r.lo, max(r.hi, 0) & ~15);
  const int tiles = r.hi > r.lo ? (r.hi - r.lo + TT - 1) / TT : 0;
  r.per_split = max(a.chunk, (tiles + a.splits - 1) / a.splits);
  r.splits = (tiles + r.per_split - 1) / r.per_split;
  return r;
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

// WD waves take the same rows and a part of the head's values each: they work out the same scores (the first product is
// theirs in full) and sum their part of V. LARGE_CAP: scores under a cap past kExpCap.
template <typename E, int D, int WR, int WK, int WD, int NST, bool LARGE_CAP>
__global__ __launch_bounds__(64 * WR * WK * WD, WK == 2 ? 1 : 2) void attention_kernel(AttnArgs a) {
  static_assert(WR == 1 || WK == 1, "waves share a tile of keys or have their own");
  static_assert(WD == 1 || (WD == 2 && WR > 1), "one of two loads K, the other V");
  constexpr int R = WR * 32;                  // rows of the workgroup
  constexpr int TT = WR > 1 ? 16 * WR : 32;   // positions of a tile
  constexpr int NS = TT / 32;                 // 32-position parts of a tile
  constexpr int GR = TT / 16 / WR;            // 16-position granules that a wave loads
  constexpr int P = kPitch<D>;
  constexpr int KS = D / 16, DT = D / 32 / WD;  // steps of the first product, a wave's 32-wide parts of the second
  constexpr int kGran = 16 * P;               // LDS bytes of a granule
  constexpr int IPG = kGran / 1024;           // loads of a granule
  constexpr int kTileB = TT * P;              // of a tile of K or of V
  constexpr int kStage = 2 * kTileB;
  constexpr int LPT = 2 / WD * GR * IPG;      // a wave's loads for a tile
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = int(threadIdx.x), lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = WR > 1 ? wave % WR : 0, wk = WR > 1 ? 0 : wave, wd = WD > 1 ? wave / WR : 0;

  // neighbouring workgroups take different key heads, so that one head's keys stay in one XCD's L2; the last rows of a
  // sequence, which see the most keys, go first
  const int id = int(gridDim.x) - 1 - int(blockIdx.x);
  const int kvh = id % a.kv_heads;
  const int rest = id / a.kv_heads;
  const int z = rest % a.splits;
  const RowTile t = row_tile<R>(a, rest / a.splits);
  if (t.rows <= 0) return;
  const int last_row = t.row0 + min(t.rows, R) - 1;
  const int pos_first = t.seq.base + t.row0 / a.group, pos_last = t.seq.base + last_row / a.group;
  const KeyRange range = key_range<TT>(a, pos_first, pos_last);
  const int tile_first = z * range.per_split;
  const bool none = z > 0 && z >= range.splits;
  if (none) return;  // the join reads as many parts as hold keys
  const int key0 = range.lo + tile_first * TT;
  const int key_end = z + 1 < range.splits ? key0 + range.per_split * TT : max(range.hi, key0);
  const int tiles = (key_end - key0 + TT - 1) / TT;  // of the workgroup; this wave: wk, wk + WK, ...

  // ---- this lane's row: row (lane & 31) of the wave's 32; rows past the last repeat it ----
  int pos;
  u32x4 qf[KS];
  {
    const int row = min(t.row0 + wr * 32 + (lane & 31), last_row);
    const int token = row / a.group, head = kvh * a.group + (row - token * a.group);
    pos = t.seq.base + token;
    if (pos >= a.capacity) pos = -1;  // no valid position: sees nothing
    const long long src = (t.seq.first + token) * a.q_stride + head * D;
    if constexpr (WR == 1) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = load_16_bytes(a.q + src + (2 * ks + half) * 8);
    } else {  // whole rows, 16 bytes for each lane; they go through LDS below (WD waves: a part of the rows each)
#pragma unroll
      for (int j = 0; j < KS / WD; ++j) {
        const int piece = (j + wd * (KS / WD)) * 64 + lane, row_of = piece / (D / 8);
        const unsigned lo = unsigned(__shfl(int(src), row_of)), hi = unsigned(__shfl(int(src >> 32), row_of));
        qf[j] = load_16_bytes(a.q + (long long)((unsigned long long)hi << 32 | lo) + piece % (D / 8) * 8);
      }
    }
  }
  const int wave_first = min(t.row0 + wr * 32, last_row), wave_last = min(t.row0 + (wr + 1) * 32 - 1, last_row);
  const int wpos_first = t.seq.base + wave_first / a.group, wpos_last = t.seq.base + wave_last / a.group;

  // ---- loads: granule g of a tile, instruction i covers 1024 / P rows ----
  constexpr int RI = 1024 / P, VP = RI < 4 ? 4 / RI : 1;  // rows of a load; loads after which V's permutation repeats
  int k_off[IPG], v_off[VP];
#pragma unroll
  for (int i = 0; i < IPG; ++i) {
    const int row = i * RI + lane / (P / 16), slot = lane % (P / 16);
    const int kc = slot ^ k_swizzle<D>(row), vc = slot ^ v_swizzle<D>(row);
    k_off[i] = kc < D / 8 ? row * 2 * D + kc * 16 : kOut;
    if (i < VP) v_off[i] = vc < D / 8 ? row * 2 * D + vc * 16 : kOut;
  }
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds) + unsigned(wk * NST * kStage));
  const const_int* table = (const const_int*)(uintptr_t)(a.page_table + (long long)t.seq.index * a.max_pages);
  int page[GR], slot16[GR];  // of the granules that the next issue() loads
  // uniform by construction; readfirstlane states it for the compiler
  const auto uniform = [](v4i r) {
    return v4i{__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y),
               __builtin_amdgcn_readfirstlane(r.z), __builtin_amdgcn_readfirstlane(r.w)};
  };
  const auto look_up = [&](int tile) {
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const int gran = min((key0 >> 4) + tile * (TT / 16) + (WR > 1 ? wr : g), (a.capacity >> 4) - 1);
      const int pg = div_magic(gran, a.page_magic, a.page_shift);
      page[g] = table[__builtin_amdgcn_readfirstlane(pg)];
      slot16[g] = gran - pg * a.page16;
    }
  };
  const auto issue = [&](int tile, int stage) {
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const int gi = WR > 1 ? wr : g;
      const int at = key0 + tile * TT + gi * 16;
      const bool there = page[g] >= 0 && page[g] < a.num_pages;
      const int bytes = there ? min(max(key_end - at, 0), 16) * 2 * D : 0;
      const long long off =
          (((long long)(there ? page[g] : 0) * a.kv_heads + kvh) * a.page16 + slot16[g]) * (16ll * 2 * D);
      v4i rk = uniform(make_vsharp(reinterpret_cast<const char*>(a.k_pages) + off, bytes));
      v4i rv = uniform(make_vsharp(reinterpret_cast<const char*>(a.v_pages) + off, bytes));
      // a vector instruction may have written these scalar registers: loads may read them 5 cycles later
      asm volatile("s_nop 4" : "+s"(rk), "+s"(rv));
      const unsigned to = lds0 + unsigned(stage * kStage + gi * kGran);
      if (WD == 1 || wd == 0)
#pragma unroll
        for (int i = 0; i < IPG; ++i) dma16(rk, to + i * 1024, k_off[i]);
      if (WD == 1 || wd == 1)
#pragma unroll
        for (int i = 0; i < IPG; ++i) dma16(rv, to + kTileB + i * 1024, v_off[i % VP] + i / VP * VP * RI * 2 * D);
    }
  };

  // ---- fragment addresses ----
  const int sl = lane & 15, g16 = lane >> 4;
  const unsigned k_rd = lds0 + unsigned((lane & 31) * P + ((half ^ k_swizzle<D>(lane & 15)) << 4));
  const unsigned v_row = unsigned(4 * half + (sl >> 2));
  const unsigned v_chunk = unsigned((2 * (g16 & 1) + ((sl & 3) >> 1)) ^ v_swizzle<D>(sl >> 2));
  const unsigned v_rd = (lds0 + unsigned(kTileB) + v_row * P + (v_chunk << 4) + ((sl & 1) << 3)) ^ unsigned(wd * DT * 64);

  // Weights are 2^(score - mc), rounded to the storage type. FP16 has no step under 2^-24, which the small weights of a
  // long cache reach: they are lifted, so that the largest lies in 2^7 .. 2^15 and one of 2^-25 of it keeps 6 bits.
  // Without the lift 131072 keys of 2^-25.2 each beside one of 1 lose their share of 0.3 % (at the same time for a call).
  constexpr float kLift = E::kDtype == GIE_HIP_FP16 ? 7.f : 0.f;
  f32x16 o[DT] = {};
  float m, mc, l;  // running maximum of the products, its power of 2 less kLift (0 while there is none), sum
  m = -INFINITY, mc = 0.f, l = 0.f;

  const auto compute = [&](int tile, int stage) {
    const unsigned so = unsigned(stage * kStage);
    const int at0 = key0 + tile * TT;
    // A value that is not finite must not reach rows that do not see its position (0 times it is a NaN): where rows of
    // the workgroup see different keys of this tile, such values are added to the rows that see them and replaced by 0.
    if ((at0 + TT - 1 > pos_first && pos_first != pos_last) || (a.window > 0 && at0 <= pos_last - a.window)) {
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < kTileB / 1024 / (WR * WD); ++i) {
        const int piece = i * WR * WD + (WR > 1 ? wave : 0);
        const u32x4 v = *reinterpret_cast<const lds_v4*>(size_t(lds0 + so + unsigned(kTileB + piece * 1024 + lane * 16)));
        bad |= not_finite<E>(v.x) | not_finite<E>(v.y) | not_finite<E>(v.z) | not_finite<E>(v.w);
      }
      bool any = __any(bad != 0);
      if constexpr (WR > 1) {  // waves that share the tile looked at a part of it each
        lds_i* found = reinterpret_cast<lds_i*>(size_t(lds0 + unsigned(NST * kStage)));
        if (lane == 0) found[wave] = any;
        stage_barrier();
        any = false;
#pragma unroll
        for (int w = 0; w < WR * WD; ++w) any |= __builtin_amdgcn_readfirstlane(found[w]) != 0;
      }
      if (any) {
        for (int k = 0; k < TT; ++k) {
          const int key = at0 + k;
          const unsigned row = lds0 + so + unsigned(kTileB + k * P);
          const uint32_t sees = key <= pos && (a.window == 0 || key > pos - a.window) ? ~0u : 0u;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int dim = 32 * (wd * DT + d) + 8 * i + 4 * half;  // 4 of them
              const u32x2 v = *reinterpret_cast<const lds_v2*>(
                  size_t(row + unsigned((((dim >> 3) ^ v_swizzle<D>(k)) << 4) + (dim & 4) * 2)));
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t word = e < 2 ? v.x : v.y;
                const uint32_t odd = 0u - ((not_finite<E>(word) >> (e & 1 ? 31 : 15)) & 1u);
                const uint32_t value = __float_as_uint(E::to_f32(uint16_t(e & 1 ? word >> 16 : word))) & odd;
                o[d][4 * i + e] += __uint_as_float(value & sees);
              }
            }
        }
        if (WR > 1) stage_barrier();
        for (int c = (WR > 1 ? tid : lane); c < kTileB / 16; c += WR * WD * 64) {
          lds_v4* at16 = reinterpret_cast<lds_v4*>(size_t(lds0 + so + unsigned(kTileB + c * 16)));
          u32x4 v = *at16;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t f = not_finite<E>(v[e]);
            v[e] &= ~((f >> 15 & 1 ? 0xffffu : 0u) | (f >> 31 ? 0xffff0000u : 0u));
          }
          *at16 = v;
        }
        if (WR > 1)
          stage_barrier();
        else
          __builtin_amdgcn_s_waitcnt(0xc07f);
      }
    }

    // Part by part of 32 keys. What a product reads from LDS is requested ahead of it: half of V under the softmax, the
    // other half and the next part's K under the second product.
    constexpr bool kAhead = WD == 1;  // where the registers hold it, or little else waits (narrow, bytes bound)
    u32x4 kf[KS];
    const auto read_k = [&](int n) {
      unsigned ko = k_rd + so;
      asm volatile("" : "+v"(ko));  // the permuted addresses are worked out for every part: kept, they cost registers
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[ks] = *reinterpret_cast<const lds_v4*>(size_t((ko ^ unsigned(ks * 32)) + unsigned(n * 32 * P)));
    };
    if (kAhead) read_k(0);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int at = at0 + n * 32;
      // scores: register i holds key at + 8 (i / 4) + 4 half + i % 4
      f32x16 s;
      s = f32x16{};
      if constexpr (kAhead) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = E::mfma32(kf[ks], qf[ks], s);
      } else {  // four steps ahead; left to itself the compiler waits for every read (one prompt
                // of 4096 at head_dim 256: 225 us, and 206 so)
        unsigned ko = k_rd + so;
        asm volatile("" : "+v"(ko));
        const auto read_4 = [&](int g) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            kf[g % 2 * 4 + i] =
                *reinterpret_cast<const lds_v4*>(size_t((ko ^ unsigned((g * 4 + i) * 32)) + unsigned(n * 32 * P)));
        };
        read_4(0);
#pragma unroll
        for (int g = 0; g < KS / 4; ++g) {
          if (g + 1 < KS / 4) read_4(g + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) s = E::mfma32(kf[g % 2 * 4 + i], qf[g * 4 + i], s);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // both halves of a part's V (16 keys each) where the registers hold them
      constexpr int VH = DT < 8 ? 2 : 1;
      u32x4 vf[VH][DT];
      const auto read_v = [&](int h) {
        unsigned vo = v_rd + so;
        asm volatile("" : "+v"(vo));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const unsigned p = (vo ^ unsigned(d * 64)) + unsigned((2 * n + h) * 16 * P);
          const u32x2 x = read_transposed(p), y = read_transposed(p + unsigned(8 * P));
          vf[h % VH][d] = u32x4{x.x, x.y, y.x, y.y};
        }
      };
      if (VH == 2) read_v(0);
      if constexpr (LARGE_CAP)
        cap_products(a, s);
      else if (a.cap > 0)
        cap_scores(a, s);
      const bool masked =
          at + 31 > wpos_first || (a.window > 0 && at <= wpos_last - a.window) || wpos_last >= a.capacity;
      if (masked) {
        const int oldest = a.window > 0 ? pos - a.window : -1;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = at + 8 * (i / 4) + 4 * half + i % 4;
          s[i] = key <= pos && key > oldest ? s[i] : -INFINITY;
        }
      }
      u32x4 pf[2];
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      top = swap_max(top);
      // the maximum follows only when a weight would pass 2^8: sums and weights keep their relative precision, and
      // most tiles leave O as it is
      if (__any((top - m) * a.mult > 8.f)) {
        const float next = fmaxf(m, top);
        float nc = next == -INFINITY ? 0.f : next * a.mult;
        // what rounding takes from nc would come on top of the lift, so 2^-23 of it is added, which is no less
        if constexpr (kLift > 0) nc += __builtin_fmaf(fabsf(nc), 0x1p-23f, -kLift);
        const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - nc);  // 1: nothing summed yet
        m = next;
        mc = nc;
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= keep;
      }
      float sum[4] = {};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.mult, -mc));
        sum[i % 4] += s[i];
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pf[h] = u32x4{E::pack2(s[8 * h], s[8 * h + 1]), E::pack2(s[8 * h + 2], s[8 * h + 3]),
                      E::pack2(s[8 * h + 4], s[8 * h + 5]), E::pack2(s[8 * h + 6], s[8 * h + 7])};
      if (VH == 2) {
        read_v(1);
        if (kAhead && n + 1 < NS) read_k(n + 1);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (VH == 1) read_v(h);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = E::mfma32(vf[h % VH][d], pf[h], o[d]);
      }
    }
  };

  // ---- main loop: a wave's j-th tile from stage j % NST while the next NST - 1 load. Loads past the last tile read
  // nothing and write zeros, so that every wait counts the same ----
  const int mine = WR > 1 ? tiles : (tiles - wk + WK - 1) / WK;
  const auto tile_at = [&](int j) { return WR > 1 ? j : wk + j * WK; };
  look_up(tile_at(0));
#pragma unroll
  for (int j = 0; j < NST - 1; ++j) {
    issue(tile_at(j), j);
    look_up(tile_at(j + 1));
  }
  if constexpr (WR > 1) {  // rows of q to the lanes that multiply them, by way of the stage that is loaded last
    static_assert(WR * 32 * P <= kStage, "the rows fit a stage");
    const unsigned rows = lds0 + unsigned((NST - 1) * kStage + wr * 32 * P);
#pragma unroll
    for (int j = 0; j < KS / WD; ++j) {
      const int piece = (j + wd * (KS / WD)) * 64 + lane, row = piece / (D / 8), c = piece % (D / 8);
      *reinterpret_cast<lds_v4*>(size_t(rows + unsigned(row * P + ((c ^ k_swizzle<D>(row & 15)) << 4)))) = qf[j];
    }
    if (WD > 1)
      stage_barrier();
    else
      __builtin_amdgcn_s_waitcnt(0xc07f);
    const unsigned mine = rows + unsigned((lane & 31) * P + ((half ^ k_swizzle<D>(lane & 15)) << 4));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const lds_v4*>(size_t(mine ^ unsigned(ks * 32)));
  }
  if (a.negate) {  // first use of q: it arrives under the loads above
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[ks][e] ^= 0x80008000u;
  }
  int stage = 0;
  for (int j = 0; j < mine; ++j) {
    wait_vm<(NST - 2) * LPT>();
    if (WR > 1)
      stage_barrier();
    else
      __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of the stage that is loaded next are done: lgkmcnt(0)
    issue(tile_at(j + NST - 1), stage == 0 ? NST - 1 : stage - 1);
    look_up(tile_at(j + NST));
    compute(tile_at(j), stage);
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
  wait_vm<0>();

  l = swap_add(l);

  // where the lane's rows go, worked out again here: kept from above it would cost registers in the loop
  int row_first = t.row0;
  asm volatile("" : "+s"(row_first));
  const auto place = [&](int& token, int& head) {
    const int row = min(row_first + wr * 32 + (lane & 31), last_row), i = row / a.group;
    token = t.seq.first + i;
    head = kvh * a.group + (row - i * a.group);
  };

  // ---- the waves' parts of the keys ----
  if constexpr (WK > 1) {
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);  // [wave][32] m, l; then [wave][32 rows][D + 4]
    if (half == 0) {
      sums[(wave * 32 + lane) * 2] = m == -INFINITY ? -INFINITY : mc;
      sums[(wave * 32 + lane) * 2 + 1] = l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) top = fmaxf(top, sums[(w * 32 + (lane & 31)) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float other = sums[(w * 32 + (lane & 31)) * 2];
      // a wave without a maximum may hold a NaN all the same
      total += sums[(w * 32 + (lane & 31)) * 2 + 1] * __builtin_amdgcn_exp2f(other == -INFINITY ? 0.f : other - ref);
    }
    const float keep = __builtin_amdgcn_exp2f(m == -INFINITY ? 0.f : mc - ref);
    constexpr int kRow = D + 4;
    float* mine_o = reinterpret_cast<float*>(lds + WK * 256) + (wave * 32 + (lane & 31)) * kRow;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(mine_o + 32 * d + 8 * i + 4 * half) =
            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * keep;
    // row (tid & 31) of the sums: every wave joins a part of the values
    m = top;
    mc = ref;
    l = total;
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(lds + WK * 256);
    const int row = lane & 31;
    if (row < t.rows) {
      int token, head;
      place(token, head);
      const float inv = total == 0.f ? 0.f : 1.f / total;
      for (int d = (wave * 2 + half) * 4; d < D; d += WK * 8) {
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < WK; ++w) v += *reinterpret_cast<const f32x4*>(all + (w * 32 + row) * kRow + d);
        if (range.splits > 1) {
          float* dst = a.part + (((long long)token * a.q_heads + head) * a.splits + z) * (D + 4);
          *reinterpret_cast<f32x4*>(dst + d) = v;
          if (d == 0) dst[D] = top, dst[D + 1] = total;
        } else {
          uint16_t* dst = a.out + token * a.o_stride + head * D + d;
          if (total == 0.f) v = f32x4{};
          v *= inv;
          store_8_bytes(dst, u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])});
        }
      }
    }
    return;
  }

  // ---- rows to out, or to the parts that are joined: through LDS, so that a store covers whole lines of a row (from
  // where the products leave them, 8 bytes of 32 rows at a time: 3.3 us longer at head_dim 256, 1.3 at 128) ----
  __syncthreads();  // the stages are free
  constexpr int kRowB = DT * 64, kPad = kRowB + 16, kPadF = 128 + 16;  // a wave's part of a row; 32 FP32 values of one
  const unsigned mine_rows = lds0 + unsigned(wave * 32 * kPad);
  const int rl = lane & 31;
  const bool there = wr * 32 + rl < t.rows;
  int token, head;
  place(token, head);
  const bool parts = range.splits > 1;
  const long long to = !there  ? -1
                       : parts ? (((long long)token * a.q_heads + head) * a.splits + z) * (D + 4) + wd * DT * 32
                               : token * a.o_stride + head * D + wd * DT * 32;
  const unsigned row = mine_rows + unsigned(rl * (parts ? kPadF : kPad));
  if (half == 0) *reinterpret_cast<lds_ll*>(size_t(row + unsigned(parts ? 128 : kRowB))) = to;
  if (parts) {
    if (there && half == 0 && wd == 0) {
      a.part[to + D] = m == -INFINITY ? -INFINITY : mc;
      a.part[to + D + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<lds_f4*>(size_t(row + unsigned((8 * i + 4 * half) * 4))) =
            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      __builtin_amdgcn_s_waitcnt(0xc07f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned from = mine_rows + unsigned((j * 8 + lane / 8) * kPadF);
        const long long at = *reinterpret_cast<const lds_ll*>(size_t(from + 128u));
        const f32x4 v = *reinterpret_cast<const lds_f4*>(size_t(from + unsigned(lane % 8 * 16)));
        if (at >= 0) *reinterpret_cast<f32x4*>(a.part + at + d * 32 + lane % 8 * 4) = v;
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 v = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (l == 0.f) v = f32x4{};  // nothing seen (and what was summed for it may be a NaN)
        v *= inv;
        *reinterpret_cast<lds_v2*>(size_t(row + unsigned((32 * d + 8 * i + 4 * half) * 2))) =
            u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
      }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    constexpr int kPieces = kRowB / 16;
#pragma unroll
    for (int j = 0; j < kPieces / 2; ++j) {
      const int piece = j * 64 + lane, from_row = piece / kPieces, c = piece % kPieces;
      const unsigned from = mine_rows + unsigned(from_row * kPad);
      const long long at = *reinterpret_cast<const lds_ll*>(size_t(from + unsigned(kRowB)));
      const u32x4 v = *reinterpret_cast<const lds_v4*>(size_t(from + unsigned(c * 16)));
      if (at >= 0) store_16_bytes(a.out + at + c * 8, v);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
}

// Joins the parts of the keys: WAVES waves for each row (token, head), lanes over the head's values 4 at a time, the parts
// dealt out to the groups of lanes that this leaves. One wave (4 rows to a workgroup) where there are few parts and many
// rows, four where one row has dozens of parts.
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

// ---- launch shape: the same on both sides of the workspace query ----
struct Shape {
  bool wide;  // rows of a workgroup: 128 that share tiles of 64 keys, or 32 with tiles of 32 for each wave
  int slots, splits, chunk;
};

constexpr int kNarrowRows = 32, kWideRows = 128, kNarrowKeys = 32, kWideKeys = 64;  // a tile's

Shape shape_of(const gie_paged_geom& g) {
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
  if (g.window > 0 && (long long)g.window + most_new < len) len = g.window + most_new;
  const long long tiles = (len + tt - 1) / tt;
  const long long blocks = busy * g.kv_heads;
  const int fewest = s.wide ? 2 : 8;  // tiles of a part
  const long long most = tiles / fewest > 1 ? tiles / fewest : 1;
  long long splits = 1;
  if (!s.wide) {
    // bytes bound: one workgroup for each compute unit, whose LDS holds 64 KiB and more on their way
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

template <typename K>
int start(K kernel, int grid, int threads, int lds_bytes, hipStream_t stream, const AttnArgs& a) {
  const int rc = set_lds_limit(reinterpret_cast<const void*>(kernel), lds_bytes);
  if (rc != GIE_HIP_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(unsigned(threads)), unsigned(lds_bytes), stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

template <typename E, int D, bool LARGE_CAP>
int launch(const AttnArgs& a, const Shape& s, hipStream_t stream) {
  const long long grid = (long long)s.slots * s.splits * a.kv_heads;
  const long long rows = (long long)a.total_tokens * a.q_heads;
  const bool many = s.splits > 8;
  const long long joining = s.splits == 1 ? 0 : many ? rows * 256 : rows * 64;
  if (grid * 512 > 0xffffffffll || joining > 0xffffff00ll) return GIE_HIP_EUNSUPPORTED;  // a launch's threads
  constexpr int P = kPitch<D>;
  int rc;
  if (s.wide) {
    constexpr int NST = 2;
    constexpr int WR = kWideRows / 32, WD = D == 256 ? 2 : 1;
    constexpr int bytes = NST * 2 * 16 * WR * P + 64;
    rc = start(attention_kernel<E, D, WR, 1, WD, NST, LARGE_CAP>, int(grid), 64 * WR * WD, bytes, stream, a);
  } else {
    constexpr int WK = D == 256 ? 2 : 4, NST = D == 64 ? 4 : 2;
    constexpr int bytes = WK * NST * 2 * 32 * P, join = WK * 256 + WK * 32 * (D + 4) * 4;
    rc = start(attention_kernel<E, D, 1, WK, 1, NST, LARGE_CAP>, int(grid), 64 * WK, bytes > join ? bytes : join, stream, a);
  }
  if (rc != GIE_HIP_OK || s.splits == 1) return rc;
  const auto join =
      s.wide ? (many ? join_kernel<E, D, kWideRows, kWideKeys, 4> : join_kernel<E, D, kWideRows, kWideKeys, 1>)
             : (many ? join_kernel<E, D, kNarrowRows, kNarrowKeys, 4> : join_kernel<E, D, kNarrowRows, kNarrowKeys, 1>);
  hipLaunchKernelGGL(join, dim3(unsigned(many ? rows : (rows + 3) / 4)), dim3(256), 0, stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

template <typename E, bool LARGE_CAP>
int launch(const AttnArgs& a, const Shape& s, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch<E, 64, LARGE_CAP>(a, s, stream);
    case 96: return launch<E, 96, LARGE_CAP>(a, s, stream);
    case 128: return launch<E, 128, LARGE_CAP>(a, s, stream);
    default: return launch<E, 256, LARGE_CAP>(a, s, stream);
  }
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_paged_attention_workspace(const gie_paged_geom* g) {
  if (!valid_paged(g) || g->total_tokens == 0) return 0;
  const Shape s = shape_of(*g);
  if (s.splits == 1) return 0;
  return size_t(g->total_tokens) * g->q_heads * s.splits * (g->head_dim + 4) * sizeof(float);
}

extern "C" int gie_hip_paged_attention(int dtype, const gie_paged_geom* g, const void* q, const void* k_pages,
                                       const void* v_pages, const int* q_starts, const int* seq_lens,
                                       const int* page_table, void* out, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  // (a scale of 0 times a masked score is a NaN)
  if (!std::isfinite(g->scale) || g->scale == 0 || !std::isfinite(g->softcap)) return GIE_HIP_EINVAL;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!q || !k_pages || !v_pages || !q_starts || !seq_lens || !page_table || !out || q == out) return GIE_HIP_EINVAL;
  if (!aligned_to(q, 2) || !aligned_to(out, 2) || !aligned_to(k_pages, 16) || !aligned_to(v_pages, 16))
    return GIE_HIP_EINVAL;
  const size_t need = gie_hip_paged_attention_workspace(g);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return GIE_HIP_EINVAL;
  const Shape shape = shape_of(*g);
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k_pages = static_cast<const uint16_t*>(k_pages);
  a.v_pages = static_cast<const uint16_t*>(v_pages);
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = g->head_dim;
  if (dtype == GIE_HIP_FP16) return large_cap ? launch<Fp16, true>(a, shape, D, s) : launch<Fp16, false>(a, shape, D, s);
  return large_cap ? launch<Bf16, true>(a, shape, D, s) : launch<Bf16, false>(a, shape, D, s);
}
