// Attention of new tokens over a paged key/value cache held in 8 bits:
//   out[t][h] = sum_j p_j vs_j c^v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * ks_j * q[t][h] . c^k_j
// (or softcap * tanh(s_j / softcap)) with codes c and the scales ks, vs of position j's block of 16, over the positions
// j <= p (and j > p - window or j < sinks), in one pass over the keys.
//
// Rows, tiles, parts and both products are those of paged_attention: 32x32x16 MFMAs with the rows in the columns. Here
// everything is FP16 in them, whatever the tokens' type: codes are exact in it, and a row of q is under a power of 2 of its
// own that puts its largest value into 2^14 .. 2^15, so that what it rounds away is under 2^-39 of that one.
//
// Scales. A block of 16 positions is half of the 32 scores that a lane has, so its scales are two constants of 8
// registers: ks is a factor of the exponent, vs a term of it, x_j = s_j log2(e) + log2(vs_j). The weight 2^(x_j - m) that
// the second product takes has vs in it, and m is the maximum of x: weights keep their bits however much the blocks'
// sizes differ. The sum of p_j takes 1 / vs once for each block.
//
// Few rows: one token over 65536 positions of 8 key heads of 128 in 32 parts 27 us (134 MB, 5.0 TB/s) + 4 for the join; a
// step of 64 sequences of 1 to 8001 120 us, 4.3 TB/s (a large copy 4.7). Many rows: two prompts of 4096 tokens, 32 heads of
// 128, 322 to 343 us by the card, 0.80 to 0.84 PFLOP/s (a large library product 1.2), where paged_attention over 16 bits
// takes 293 to 311. The vector unit is busy 0.61 of the time and the matrix cores 0.39, one after the other whatever was
// tried: codes decoded under matrix instructions, scores of the next part under the weights (2 %, kept), wave priorities;
// so what helps is fewer vector instructions. Of the 240 that a wave has for a tile of 64 keys, and 32 exponentials at a
// quarter of their rate, 80 decode and 80 are the weights, their sum and their rounding. 256 rows that share a tile (half
// the decoding for each) took from 8 % less (one prompt) to 30 % more (ragged ones, narrow heads).
// Outputs are off by 1.7e-3 of their size in BF16, as FP32 weights with one rounding would be: FP16's rounding of the
// weights is small beside it. In FP16 it is not: 2.2e-4 over long contexts, up to 3.1e-4 over short ones (1.4 times the
// FP32 form).
#include <type_traits>

#include "attention_common.h"
#include "kv8_common.h"

namespace gie_hip {
namespace {

typedef __attribute__((address_space(3))) float lds_float;

struct Kv8Args : AttnArgs {
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scales;
  const float* v_scales;
  unsigned page_blocks;  // blocks of a page of all key heads
  int bf16;              // type of q and out
};

constexpr float kLift = 7.f;  // weights lie in 2^7 .. 2^15 at their largest: FP16 has no step under 2^-24

// A block's scales as the scores take them: f times the product of codes and the row's factor is the score's power of 2,
// or where scores are capped the product of keys (a NaN if either scale is one: every score of the block becomes a NaN),
// lv = log2(vs), inv = 1 / vs. The codes' unit is in the row's factor: the largest scale times it passes FP32's range.
struct BlockScales {
  float f, lv, inv;
};
__device__ __forceinline__ BlockScales block_scales(const AttnArgs& a, float ks, float vs) {
  // (int8's scale of the largest FP32 value lies just above 2^121)
  const float k = fminf(fmaxf(ks, 0x1p-73f), 0x1p122f), v = fminf(fmaxf(vs, 0x1p-73f), 0x1p122f);
  const bool bad = !(ks == ks) || !(vs == vs);
  // the exponent and the quotient from the same logarithm, so that a weight and what the sum takes of it agree
  const float lv = __builtin_amdgcn_logf(v);
  return {bad ? __builtin_nanf("") : k * (a.cap > 0 ? 1.f : a.mult), lv, __builtin_amdgcn_exp2f(-lv)};
}

// A block of a sequence as a lane finds it: where it lies among all blocks (kNoBlock: its page is not there, its codes
// count as zeros), and its scales.
constexpr unsigned kNoBlock = 0xffffffffu;
struct BlockAt {
  unsigned at;
  BlockScales s;
};
// The lanes look up 64 blocks at once, and the loop takes them by readlane: loads through the scalar cache would share
// their counter with LDS, so that every wait for a fragment waited for them.
__device__ __forceinline__ BlockAt find_block(const Kv8Args& a, const int* table, int kvh, int position) {
  const int gran = min(position >> 4, (a.capacity >> 4) - 1), pg = div_magic(gran, a.page_magic, a.page_shift);
  const int page = table[pg];
  const bool there = unsigned(page) < unsigned(a.num_pages);
  BlockAt b;
  b.at = there ? unsigned(page) * a.page_blocks + unsigned(kvh * a.page16 + gran - pg * a.page16) : kNoBlock;
  b.s = block_scales(a, there ? a.k_scales[b.at] : 0.f, there ? a.v_scales[b.at] : 0.f);
  return b;
}
__device__ __forceinline__ float read_lane(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
__device__ __forceinline__ BlockAt block_of_lane(const BlockAt& b, int lane) {
  return {unsigned(__builtin_amdgcn_readlane(int(b.at), lane)),
          {read_lane(b.s.f, lane), read_lane(b.s.lv, lane), read_lane(b.s.inv, lane)}};
}

// codes of 8 values, in the order 0, 2, 1, 3, 4, 6, 5, 7
template <typename C>
__device__ __forceinline__ u32x4 decode8(uint32_t a, uint32_t b) {
  const u32x2 x = C::decode4(a), y = C::decode4(b);
  return u32x4{x.x, x.y, y.x, y.y};
}

// Fragments of a row of q (this lane's half of its values) in FP16, in decode8's order, times a power of 2; returns the
// factor that takes it back. The sign changes where the scores' scale is negative.
template <typename E, int KS>
__device__ __forceinline__ float row_to_fp16(u32x4 (&qf)[KS], bool negate) {
  const auto value = [&](int ks, int i) { return E::to_f32(uint16_t(qf[ks][i / 2] >> (i % 2 * 16))); };
  float most = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(value(ks, i)));
  most = swap_max(most);
  const int e = max(int(__float_as_uint(most) >> 23) - 127, -100);
  float f = __uint_as_float(unsigned(127 + 14 - e) << 23);
  if (negate) f = -f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = Fp16::pack2(value(ks, 4 * i) * f, value(ks, 4 * i + 2) * f);
      r[2 * i + 1] = Fp16::pack2(value(ks, 4 * i + 1) * f, value(ks, 4 * i + 3) * f);
    }
    qf[ks] = r;
  }
  return __uint_as_float(unsigned(127 + e - 14) << 23);
}

__device__ __forceinline__ u32x2 pack_out(bool bf16, f32x4 v) {
  if (bf16) return u32x2{Bf16::pack2(v[0], v[1]), Bf16::pack2(v[2], v[3])};
  return u32x2{Fp16::pack2(v[0], v[1]), Fp16::pack2(v[2], v[3])};
}

// The weights of 32 scores (register i: key 8 (i / 4) + 4 half + i % 4, so the block i / 8), and what they do to the
// running maximum, the sum and the rows' values. `masked`: seen(i) says whether register i's key is.
//
// The maximum is not looked for ahead of the weights (which took 27 of about 150 vector instructions, and 8 % of the time
// of two prompts of 4096): they are taken against what is there, and as long as a lane's sum of them stays within 2^15 all
// of them fit FP16. Only where it does not, or a row has seen nothing yet, the rows' maxima move and the weights are taken
// again.
template <bool LARGE_CAP, typename Seen>
__device__ __forceinline__ void cap_and_mask(const AttnArgs& a, f32x16& s, const BlockScales (&sc)[2], float row_factor,
                                             bool masked, Seen seen, float (&f)[2]) {
  const auto within = [](float x) { return __builtin_amdgcn_fmed3f(x, 0x1p-126f, 3e38f); };  // masked: no -inf times 0
  f[0] = within(row_factor * sc[0].f);
  f[1] = within(row_factor * sc[1].f);
  if (LARGE_CAP || a.cap > 0) {
    if constexpr (LARGE_CAP) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= f[i / 8];
      cap_products(a, s);
    } else {  // cap_scores with the block's factor in the exponent's
      const float in[2] = {fminf(f[0] * a.cap_in, 3e38f), fminf(f[1] * a.cap_in, 3e38f)};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[i] * in[i / 8]);
        s[i] = a.cap - 2.f * a.cap * __builtin_amdgcn_rcpf(e + 1.f);
      }
    }
    f[0] = f[1] = a.mult;
  }
  if (__any(!(sc[0].f == sc[0].f) || !(sc[1].f == sc[1].f))) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
      if (!(sc[g].f == sc[g].f)) {
        f[g] = 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[8 * g + i] = __builtin_nanf("");
      }
  }
  if (masked) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = seen(i) ? s[i] : -INFINITY;
  }
}
struct Weights {
  f32x16 w;
  float c[2], sum[2][2];
  __device__ __forceinline__ void begin(const BlockScales (&sc)[2], float mc) { c[0] = sc[0].lv - mc, c[1] = sc[1].lv - mc; }
  __device__ __forceinline__ void take(const f32x16& s, const float (&f)[2], int i) {
    const int g = i / 8;
    w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], f[g], c[g]));
    sum[g][i % 2] = i % 8 < 2 ? w[i] : sum[g][i % 2] + w[i];
  }
  __device__ __forceinline__ void take_all(const f32x16& s, const float (&f)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) take(s, f, i);
  }
  __device__ __forceinline__ bool overflows() const {
    return !((sum[0][0] + sum[0][1]) + (sum[1][0] + sum[1][1]) <= 0x1p15f);  // (or a NaN)
  }
  // the scores' largest exponent, the same in both halves of the wave
  __device__ __forceinline__ float top(const f32x16& s, const float (&f)[2], const BlockScales (&sc)[2]) const {
    float t = -INFINITY;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float most = s[8 * g];
#pragma unroll
      for (int i = 1; i < 8; ++i) most = fmaxf(most, s[8 * g + i]);
      t = fmaxf(t, __builtin_fmaf(most, f[g], sc[g].lv));
    }
    return swap_max(t);
  }
  // a row's maximum to what it is with `top`
  template <int DT>
  static __device__ __forceinline__ void move(float top, float& m, float& mc, float& l, f32x16 (&o)[DT]) {
    const float next = fmaxf(m, top);
    float nc = next == -INFINITY ? 0.f : next;
    nc += __builtin_fmaf(fabsf(nc), 0x1p-22f, -kLift);  // (what rounding takes from it and from an exponent)
    const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - nc);  // 1: nothing summed yet
    m = next;
    mc = nc;
    l *= keep;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= keep;
  }
  __device__ __forceinline__ void add_to(float& l, const BlockScales (&sc)[2]) const {
    l = __builtin_fmaf(sum[0][0] + sum[0][1], sc[0].inv, l);
    l = __builtin_fmaf(sum[1][0] + sum[1][1], sc[1].inv, l);
  }
  // of one block, in the order of its keys
  __device__ __forceinline__ u32x4 packed(int h) const {
    return u32x4{Fp16::pack2(w[8 * h], w[8 * h + 1]), Fp16::pack2(w[8 * h + 2], w[8 * h + 3]),
                 Fp16::pack2(w[8 * h + 4], w[8 * h + 5]), Fp16::pack2(w[8 * h + 6], w[8 * h + 7])};
  }
};
template <int DT>
__device__ __forceinline__ void settle(Weights& w, const f32x16& s, const float (&f)[2], const BlockScales (&sc)[2],
                                       float& m, float& mc, float& l, f32x16 (&o)[DT]) {
  if (__any(w.overflows() || m == -INFINITY)) {
    w.move(w.top(s, f, sc), m, mc, l, o);
    w.begin(sc, mc);
    w.take_all(s, f);
  }
  w.add_to(l, sc);
}

// ---------------------------------------------------------------- few rows: 32 for each workgroup
// Bound by the cache's bytes. Codes go HBM -> LDS by direct loads and are decoded in the registers of the wave that
// multiplies them: WK waves with tiles of 32 keys of their own and NST stages each, no barrier until they are joined. LDS
// and registers hold one workgroup for each compute unit, at head_dim 64 two (64 sequences of 4000, 8 key heads: 49 us; with
// one and four stages 58).
// K: 16 bytes of a row for two steps of the first product (the order of the summed values is free as long as q has the
// same). V: ds_read_b64_tr_b8 gives a lane 8 keys of its value. 16-byte chunks of a row are permuted by the row so that
// both reads meet no bank twice in a phase.
template <int D>
constexpr int kPitch8 = D == 96 ? 128 : D;  // bytes of a row of codes in LDS
template <int D>
__device__ __forceinline__ int k_swizzle8(int row) {
  return D == 64 ? (row >> 2) & 3 : D == 256 ? row & 15 : (row >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int v_swizzle8(int row) {
  const int far = (row >> 3) & 1;
  return D == 64 ? far * 2 : D == 256 ? (row & 3) * 2 + far * 8 : ((row >> 1) & 1) * 2 + far * 4;
}

// a 16-lane group reads 8 rows of 16 bytes; each lane gets the 8 rows' bytes of its column
__device__ __forceinline__ u32x2 read_transposed8(unsigned at) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                       reinterpret_cast<__attribute__((address_space(3))) v2i*>(size_t(at))));
}

template <typename C, int D, int WK, int NST, bool LARGE_CAP>
__global__ __launch_bounds__(64 * WK, D == 64 ? 4 : WK == 8 ? 2 : 1) void narrow_kernel(Kv8Args a) {
  constexpr int TT = kNarrowKeys, GR = TT / 16, P = kPitch8<D>, KS = D / 16, KP = D / 32, DT = D / 32;
  constexpr int kGran = 16 * P, IPG = kGran / 1024, kTileB = TT * P, kStage = 2 * kTileB, LPT = 2 * GR * IPG;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = int(threadIdx.x), lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // neighbouring workgroups take different key heads, the last rows of a sequence go first
  const int id = int(gridDim.x) - 1 - int(blockIdx.x);
  const int kvh = id % a.kv_heads, rest = id / a.kv_heads, z = rest % a.splits;
  const RowTile t = row_tile<kNarrowRows>(a, rest / a.splits);
  if (t.rows <= 0) return;
  const int last_row = t.row0 + min(t.rows, kNarrowRows) - 1;
  const int pos_first = t.seq.base + t.row0 / a.group, pos_last = t.seq.base + last_row / a.group;
  const KeyRange range = key_range<TT>(a, pos_first, pos_last);
  const int tile_first = z * range.per_split;
  if (z > 0 && z >= range.splits) return;  // the join reads as many parts as hold keys
  const int tiles = min(range.per_split, range.tiles - tile_first);  // of the workgroup; this wave: wave, wave + WK, ...
  const int turn = range.sink_tiles - tile_first, sink0 = tile_first * TT;
  const int key0 = sink0 + range.lo - range.sink_tiles * TT;
  const auto key_of = [&](int tile) { return tile * TT + (tile < turn ? sink0 : key0); };

  // ---- this lane's row: row (lane & 31); rows past the last repeat it ----
  const int row = min(t.row0 + (lane & 31), last_row);
  const int token = row / a.group, head = kvh * a.group + (row - token * a.group);
  int pos = t.seq.base + token;
  if (pos >= a.capacity) pos = -1;  // no valid position: sees nothing
  u32x4 qf[KS];
  {
    const uint16_t* src = a.q + (t.seq.first + token) * a.q_stride + head * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_16_bytes(src + 16 * (ks - ks % 2 + half) + 8 * (ks % 2));
  }

  // ---- loads: granule g of a tile, instruction i covers 1024 / P rows ----
  constexpr int RI = 1024 / P;
  int k_off[IPG], v_off[IPG];
#pragma unroll
  for (int i = 0; i < IPG; ++i) {
    const int r = i * RI + lane / (P / 16), slot = lane % (P / 16);
    const int kc = slot ^ k_swizzle8<D>(r), vc = slot ^ v_swizzle8<D>(r);
    k_off[i] = kc < D / 16 ? r * D + kc * 16 : kOut;
    v_off[i] = vc < D / 16 ? r * D + vc * 16 : kOut;
  }
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds) + unsigned(wave * NST * kStage));
  const int* table = a.page_table + (long long)t.seq.index * a.max_pages;
  const auto tile_at = [&](int j) { return wave + j * WK; };  // the wave's j-th tile
  BlockAt blocks;  // lane 2 i + g: granule g of the wave's tile j with j % 32 == i
  const auto uniform = [](v4i r) {
    return v4i{__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y),
               __builtin_amdgcn_readfirstlane(r.z), __builtin_amdgcn_readfirstlane(r.w)};
  };
  struct Pair {
    BlockScales g[GR];
  };
  // requests the wave's j-th tile
  const auto issue = [&](int j, int stage, Pair& scales) {
    if (j % 32 == 0) blocks = find_block(a, table, kvh, key_of(tile_at(j + lane / GR)) + lane % GR * 16);
    const int tile = tile_at(j);
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const BlockAt b = block_of_lane(blocks, j % 32 * GR + g);
      scales.g[g] = b.s;
      const int at = key_of(tile) + g * 16;
      const int bytes = b.at != kNoBlock && tile < tiles ? min(max(range.hi - at, 0), 16) * D : 0;
      const unsigned long long off = (b.at != kNoBlock ? b.at : 0u) * (unsigned long long)(16 * D);
      v4i rk = uniform(make_vsharp(a.k_pages + off, bytes)), rv = uniform(make_vsharp(a.v_pages + off, bytes));
      // a vector instruction may have written these scalar registers: loads may read them 5 cycles later
      asm volatile("s_nop 4" : "+s"(rk), "+s"(rv));
      const unsigned to = lds0 + unsigned(stage * kStage + g * kGran);
#pragma unroll
      for (int i = 0; i < IPG; ++i) dma16(rk, to + i * 1024, k_off[i]);
#pragma unroll
      for (int i = 0; i < IPG; ++i) dma16(rv, to + kTileB + i * 1024, v_off[i]);
    }
  };

  // ---- fragment addresses ----
  const int sl = lane & 15, chunk = (lane >> 4) & 1;
  const unsigned k_rd = lds0 + unsigned((lane & 31) * P + ((half ^ k_swizzle8<D>(lane & 15)) << 4));
  const int v_row = 4 * half + (sl >> 1 & 3) + 8 * (sl >> 3);
  const unsigned v_rd = lds0 + unsigned(kTileB + v_row * P + ((chunk ^ v_swizzle8<D>(v_row)) << 4) + (sl & 1) * 8);

  f32x16 o[DT] = {};
  float m = -INFINITY, mc = 0.f, l = 0.f;  // running maximum of the exponents, what is taken from them, sum
  float row_factor = 1.f;

  const auto compute = [&](int tile, int stage, const Pair& pair) {
    const unsigned so = unsigned(stage * kStage);
    const int at = key_of(tile), oldest = a.window > 0 ? pos - a.window : -1;
    u32x4 kr[KP];
#pragma unroll
    for (int i = 0; i < KP; ++i) kr[i] = *reinterpret_cast<const lds_v4*>(size_t((k_rd + so) ^ unsigned(i * 32)));
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      s = Fp16::mfma32(decode8<C>(kr[i].x, kr[i].y), qf[2 * i], s);
      s = Fp16::mfma32(decode8<C>(kr[i].z, kr[i].w), qf[2 * i + 1], s);
    }
    u32x2 vr[2][DT];  // requested under the weights
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[g][d] = read_transposed8(((v_rd + so) ^ unsigned(d * 32)) + unsigned(g * kGran));
    const bool masked = at + TT - 1 > pos_first || (a.window > 0 && at <= pos_last - a.window) || pos_last >= a.capacity;
    const auto seen = [&](int i) { return sees(a, at + 8 * (i / 4) + 4 * half + i % 4, pos, oldest); };
    float f[2];
    cap_and_mask<LARGE_CAP>(a, s, pair.g, row_factor, masked, seen, f);
    Weights w;
    w.begin(pair.g, mc);
    w.take_all(s, f);
    settle(w, s, f, pair.g, m, mc, l, o);
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // in decode8's order of the keys
      const f32x16& p = w.w;
      const u32x4 pf = {Fp16::pack2(p[8 * g], p[8 * g + 2]), Fp16::pack2(p[8 * g + 1], p[8 * g + 3]),
                        Fp16::pack2(p[8 * g + 4], p[8 * g + 6]), Fp16::pack2(p[8 * g + 5], p[8 * g + 7])};
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = Fp16::mfma32(decode8<C>(vr[g][d].x, vr[g][d].y), pf, o[d]);
    }
  };

  // ---- main loop: a wave's j-th tile from stage j % NST while the next NST - 1 load; loads past the last tile read
  // nothing and write zeros, so that every wait counts the same ----
  const int mine = (tiles - wave + WK - 1) / WK;
  Pair scales[NST - 1];  // of the tiles that load
#pragma unroll
  for (int j = 0; j < NST - 1; ++j) issue(j, j, scales[j]);
  row_factor = (a.bf16 ? row_to_fp16<Bf16>(qf, a.negate != 0) : row_to_fp16<Fp16>(qf, a.negate != 0)) * C::kUnit;
  int stage = 0;
  for (int j = 0; j < mine; ++j) {
    wait_vm<(NST - 2) * LPT>();
    __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of the stage that is loaded next are done: lgkmcnt(0)
    const Pair now = scales[0];
#pragma unroll
    for (int i = 0; i + 1 < NST - 1; ++i) scales[i] = scales[i + 1];
    issue(j + NST - 1, stage == 0 ? NST - 1 : stage - 1, scales[NST - 2]);
    compute(tile_at(j), stage, now);
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
  wait_vm<0>();
  l = swap_add(l);

  // ---- the waves' parts of the keys ----
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
  const float keep = __builtin_amdgcn_exp2f(m == -INFINITY ? 0.f : mc - ref) * C::kUnit;
  constexpr int kRow = D + 4;
  float* mine_o = reinterpret_cast<float*>(lds + WK * 256) + (wave * 32 + (lane & 31)) * kRow;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(mine_o + 32 * d + 8 * i + 4 * half) =
          f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * keep;
  // row (tid & 31) of the sums: every wave joins a part of the values
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(lds + WK * 256);
  const int r = lane & 31;
  if (r >= t.rows) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int d = (wave * 2 + half) * 4; d < D; d += WK * 8) {
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < WK; ++w) v += *reinterpret_cast<const f32x4*>(all + (w * 32 + r) * kRow + d);
    if (range.splits > 1) {
      float* dst = a.part + (((long long)(t.seq.first + token) * a.q_heads + head) * a.splits + z) * (D + 4);
      *reinterpret_cast<f32x4*>(dst + d) = v;
      if (d == 0) dst[D] = top, dst[D + 1] = total;
    } else {
      uint16_t* dst = a.out + (t.seq.first + token) * a.o_stride + head * D + d;
      if (total == 0.f) v = f32x4{};
      v *= inv;
      store_8_bytes(dst, pack_out(a.bf16, v));
    }
  }
}

// ---------------------------------------------------------------- many rows: 128 for each workgroup
// Bound by the products and the softmax. The workgroup decodes a tile of 64 keys once, HBM -> registers -> LDS in FP16, for
// the waves that share it: a wave decoding what it multiplies would decode every code four times. Codes of the next tile
// but one are requested before a tile is worked on. Values lie in decode8's order in LDS: of K that is q's order too, of
// V the rows' registers are put in order at the end.
// Up to head_dim 128 four waves take 32 rows each, in steps of half a tile. At 256 (WD == 2) two waves share 32 rows, for
// each has registers for half of the values; each works out half of a tile's scores, and they exchange the weights through
// LDS (512 tokens over 8192, 32 heads: 174 us; with all scores worked out by both 219).
template <typename C, int D, int WD, bool LARGE_CAP>
__global__ __launch_bounds__(256 * WD, 2) void wide_kernel(Kv8Args a) {
  constexpr int WR = kWideRows / 32, R = kWideRows, TT = kWideKeys, NS = TT / 32, P = kPitch<D>;
  constexpr int KS = D / 16, DT = D / 32 / WD, kTileB = TT * P, kStage = 2 * kTileB;
  constexpr int kPieces = D, JP = (kPieces + 63) / 64;  // 16-byte pieces of a granule's codes, of a lane
  constexpr int kConst = 2 * kStage;                    // [stage][granule] BlockScales
  // WD == 2: weights [wave][block of 16][lane], whether a wave's maxima move [wave], maxima [wave][row]
  constexpr int kExchange = kConst + 2 * WR * 16, kFlags = kExchange + 2 * WR * 2048, kTops = kFlags + 2 * WR * 4;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = int(threadIdx.x), lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % WR, wd = wave / WR;

  const int id = int(gridDim.x) - 1 - int(blockIdx.x);
  const int kvh = id % a.kv_heads, rest = id / a.kv_heads, z = rest % a.splits;
  const RowTile t = row_tile<R>(a, rest / a.splits);
  if (t.rows <= 0) return;
  const int last_row = t.row0 + min(t.rows, R) - 1;
  const int pos_first = t.seq.base + t.row0 / a.group, pos_last = t.seq.base + last_row / a.group;
  const KeyRange range = key_range<TT>(a, pos_first, pos_last);
  const int tile_first = z * range.per_split;
  if (z > 0 && z >= range.splits) return;
  const int tiles = min(range.per_split, range.tiles - tile_first);
  const int turn = range.sink_tiles - tile_first, sink0 = tile_first * TT;
  const int key0 = sink0 + range.lo - range.sink_tiles * TT;
  const auto key_of = [&](int tile) { return tile * TT + (tile < turn ? sink0 : key0); };

  int pos;
  u32x4 qf[KS];
  {
    const int row = min(t.row0 + wr * 32 + (lane & 31), last_row);
    const int token = row / a.group, head = kvh * a.group + (row - token * a.group);
    pos = t.seq.base + token;
    if (pos >= a.capacity) pos = -1;  // no valid position: sees nothing
    const long long src = (t.seq.first + token) * a.q_stride + head * D;
    // whole rows, 16 bytes for each lane; they go through LDS below (WD waves: a part of the rows each)
#pragma unroll
    for (int j = 0; j < KS / WD; ++j) {
      const int piece = (j + wd * (KS / WD)) * 64 + lane, row_of = piece / (D / 8);
      const unsigned lo = unsigned(__shfl(int(src), row_of)), hi = unsigned(__shfl(int(src >> 32), row_of));
      qf[j] = load_16_bytes(a.q + (long long)((unsigned long long)hi << 32 | lo) + piece % (D / 8) * 8);
    }
  }
  const int wave_first = min(t.row0 + wr * 32, last_row), wave_last = min(t.row0 + (wr + 1) * 32 - 1, last_row);
  const int wpos_first = t.seq.base + wave_first / a.group, wpos_last = t.seq.base + wave_last / a.group;

  // ---- codes: granule wr of a tile by this wave (of K and V, or WD == 2: of one) ----
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds));
  const int* table = a.page_table + (long long)t.seq.index * a.max_pages;
  BlockAt blocks;  // lane i: granule wr of the tile j with j % 64 == i
  constexpr int KV = 2 / WD;  // of this wave
  static_assert(NS == 2, "a half of the pieces for each part");
  // Half of a tile's pieces at a time: K's, then V's (WD == 2: two halves of the one). Pieces go under the first products
  // of one part of the tile before: decoded there they cost no time of their own.
  constexpr int kHalf = KV * JP / 2;
  u32x4 raw[2][kHalf];
  BlockAt now;
  const auto load = [&](int tile, int n) {
    if (n == 0) {
      if (tile % 64 == 0) blocks = find_block(a, table, kvh, key_of(tile + lane) + wr * 16);
      now = block_of_lane(blocks, tile % 64);
    }
    const int at = key_of(tile) + wr * 16;
    const int bytes = now.at != kNoBlock && tile < tiles ? min(max(range.hi - at, 0), 16) * D : 0;
    const unsigned long long off = (now.at != kNoBlock ? now.at : 0u) * (unsigned long long)(16 * D);
    const uint8_t* from = ((WD == 1 ? n == 1 : wd == 1) ? a.v_pages : a.k_pages) + off;
    // uniform by construction; readfirstlane states it for the compiler
    const unsigned long long address = reinterpret_cast<unsigned long long>(from);
    const unsigned lo = __builtin_amdgcn_readfirstlane(unsigned(address)), hi = __builtin_amdgcn_readfirstlane(unsigned(address >> 32));
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((unsigned long long)hi << 32 | lo), 0,
                                                        __builtin_amdgcn_readfirstlane(bytes), kBufferWord3);
#pragma unroll
    for (int j = 0; j < kHalf; ++j)
      raw[n][j] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (((WD == 1 ? 0 : n * kHalf) + j) * 64 + lane) * 16, 0, 0));
  };
  // piece j * 64 + lane: 16 values of a row, two chunks of FP16
  unsigned k_wr[JP], v_wr[JP];
#pragma unroll
  for (int j = 0; j < JP; ++j) {
    const int piece = j * 64 + lane, row = piece / (D / 16), c = piece % (D / 16) * 2;
    k_wr[j] = unsigned((wr * 16 + row) * P + ((c ^ k_swizzle<D>(row)) << 4));
    v_wr[j] = unsigned(kTileB + (wr * 16 + row) * P + ((c ^ v_swizzle<D>(row)) << 4));
  }
  // unit u of 2 kHalf: 8 values of a piece for each lane
  const auto decode_unit = [&](int n, int u, int stage) {
    const bool is_v = WD == 1 ? n == 1 : wd == 1;
    const int j = u / 2, at = (WD == 1 ? 0 : n * kHalf) + j;
    if (kPieces % 64 != 0 && at * 64 + lane >= kPieces) return;
    const unsigned to = lds0 + unsigned(stage * kStage) + (is_v ? v_wr[at] : k_wr[at]);
    const u32x4 r = raw[n][j];
    *reinterpret_cast<lds_v4*>(size_t(u % 2 ? to ^ 16u : to)) = u % 2 ? decode8<C>(r.z, r.w) : decode8<C>(r.x, r.y);
  };
  const auto store_scales = [&](int stage) {
    if (wd != 0) return;
    if (lane == 0)
      *reinterpret_cast<lds_f4*>(size_t(lds0 + unsigned(kConst + (stage * WR + wr) * 16))) =
          f32x4{now.s.f, now.s.lv, now.s.inv, 0.f};
  };

  // ---- fragment addresses ----
  const int sl = lane & 15, g16 = lane >> 4;
  const unsigned k_rd = lds0 + unsigned((lane & 31) * P + ((half ^ k_swizzle<D>(lane & 15)) << 4));
  const unsigned v_row = unsigned(4 * half + (sl >> 2));
  const unsigned v_chunk = unsigned((2 * (g16 & 1) + ((sl & 3) >> 1)) ^ v_swizzle<D>(sl >> 2));
  const unsigned v_rd = (lds0 + unsigned(kTileB) + v_row * P + (v_chunk << 4) + ((sl & 1) << 3)) ^ unsigned(wd * DT * 64);

  f32x16 o[DT] = {};
  float m = -INFINITY, mc = 0.f, l = 0.f;
  float row_factor = 1.f;

  // WD == 2: a tile by the two waves of the same rows. Each works out the scores of one part's keys and their weights; they
  // exchange the weights through LDS (and, when one of the workgroup's maxima has to move, the maxima first) and sum their
  // halves of the values over both parts. l is a wave's own part of the sum until the end.
  const auto pair_tile = [&](int tile, auto stage_of) {
    const int stage = stage_of;
    const unsigned so = unsigned(stage * kStage);
    const int at = key_of(tile) + wd * 32, oldest = a.window > 0 ? pos - a.window : -1;
    store_scales(stage ^ 1);
    f32x16 s = {};
    {
      u32x4 kf[8];
      unsigned ko = k_rd + so + unsigned(wd * 32 * P);
      asm volatile("" : "+v"(ko));  // the permuted addresses are worked out for every tile: kept, they cost registers
      const auto read_4 = [&](int g) {  // four steps ahead
#pragma unroll
        for (int i = 0; i < 4; ++i)
          kf[g % 2 * 4 + i] = *reinterpret_cast<const lds_v4*>(size_t(ko ^ unsigned((g * 4 + i) * 32)));
      };
      read_4(0);
      constexpr int kUnits = 4 * kHalf, G = KS / 4;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g + 1 < G) read_4(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = Fp16::mfma32(kf[g % 2 * 4 + i], qf[g * 4 + i], s);
#pragma unroll
        for (int u = g * kUnits / G; u < (g + 1) * kUnits / G; ++u) decode_unit(u / (2 * kHalf), u % (2 * kHalf), stage ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    load(tile + 2, 0);
    load(tile + 2, 1);
    BlockScales sc[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const f32x4 c = *reinterpret_cast<const lds_f4*>(size_t(lds0 + unsigned(kConst + (stage * WR + 2 * wd + g) * 16)));
      sc[g] = {c[0], c[1], c[2]};
    }
    // V: granules of this wave's own part first
    u32x4 vf[2][DT];
    const auto read_v = [&](int k) {
      unsigned vo = v_rd + so + unsigned((k / 2 == 0 ? wd : wd ^ 1) * 32 * P);
      asm volatile("" : "+v"(vo));
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const unsigned p = (vo ^ unsigned(d * 64)) + unsigned(k % 2 * 16 * P);
        const u32x2 x = read_transposed(p), y = read_transposed(p + unsigned(8 * P));
        vf[k % 2][d] = u32x4{x.x, x.y, y.x, y.y};
      }
    };
    read_v(0);
    const bool masked = at + 31 > wpos_first || (a.window > 0 && at <= wpos_last - a.window) || wpos_last >= a.capacity;
    const auto seen = [&](int i) { return sees(a, at + 8 * (i / 4) + 4 * half + i % 4, pos, oldest); };
    float f[2];
    cap_and_mask<LARGE_CAP>(a, s, sc, row_factor, masked, seen, f);
    Weights w;
    w.begin(sc, mc);
    w.take_all(s, f);
    u32x4 pf[2];
    const unsigned exchange = lds0 + unsigned(kExchange + lane * 16), flags = lds0 + unsigned(kFlags);
    const auto give = [&] {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pf[h] = w.packed(h);
        *reinterpret_cast<lds_v4*>(size_t(exchange + unsigned(wave * 2048 + h * 1024))) = pf[h];
      }
    };
    give();
    const bool moves = w.overflows() || m == -INFINITY;
    const int any_moves = __any(moves);
    if (lane == 0) *reinterpret_cast<lds_i*>(size_t(flags + unsigned(wave * 4))) = any_moves;
    stage_barrier();
    int all_moves = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 x = *reinterpret_cast<const lds_v4*>(size_t(flags + unsigned(i * 16)));
      all_moves |= int(x.x | x.y | x.z | x.w);
    }
    if (__builtin_amdgcn_readfirstlane(all_moves) != 0) {  // the same in all waves
      const float top = w.top(s, f, sc);
      const unsigned tops = lds0 + unsigned(kTops + (lane & 31) * 4);
      *reinterpret_cast<lds_float*>(size_t(tops + unsigned(wave * 128))) = top;
      stage_barrier();
      const float other = *reinterpret_cast<const lds_float*>(size_t(tops + unsigned((wave ^ WR) * 128)));
      w.move(fmaxf(top, other), m, mc, l, o);
      w.begin(sc, mc);
      w.take_all(s, f);
      give();
      stage_barrier();
    }
    w.add_to(l, sc);
    u32x4 of[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      of[h] = *reinterpret_cast<const lds_v4*>(size_t(exchange + unsigned((wave ^ WR) * 2048 + h * 1024)));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k < 3) read_v(k + 1);
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = Fp16::mfma32(vf[k % 2][d], k < 2 ? pf[k] : of[k - 2], o[d]);
    }
  };

  // One part of a tile, half of a tile's work: the weights of scores that are there (s), under them the scores of the part
  // after it, then the values, under them codes of the next tile.
  const auto step = [&](int tile, auto part, f32x16& s) {
    constexpr int n = decltype(part)::value;
    const int stage = tile & 1, k_stage = n == 0 ? stage : stage ^ 1;
    const int at = key_of(tile) + n * 32, oldest = a.window > 0 ? pos - a.window : -1;
    if (n == 0) store_scales(stage ^ 1);
    u32x4 kf[KS], vf[2][DT];
    {
      unsigned ko = k_rd + unsigned(k_stage * kStage + (n ^ 1) * 32 * P);
      asm volatile("" : "+v"(ko));
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[ks] = *reinterpret_cast<const lds_v4*>(size_t(ko ^ unsigned(ks * 32)));
    }
    BlockScales sc[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const f32x4 c = *reinterpret_cast<const lds_f4*>(size_t(lds0 + unsigned(kConst + (stage * WR + 2 * n + g) * 16)));
      sc[g] = {c[0], c[1], c[2]};
    }
    const auto read_v = [&](int h) {
      unsigned vo = v_rd + unsigned(stage * kStage);
      asm volatile("" : "+v"(vo));
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const unsigned p = (vo ^ unsigned(d * 64)) + unsigned((2 * n + h) * 16 * P);
        const u32x2 x = read_transposed(p), y = read_transposed(p + unsigned(8 * P));
        vf[h][d] = u32x4{x.x, x.y, y.x, y.y};
      }
    };
    const bool masked =
        at + 31 > wpos_first || (a.window > 0 && at <= wpos_last - a.window) || wpos_last >= a.capacity;
    const auto seen = [&](int i) { return sees(a, at + 8 * (i / 4) + 4 * half + i % 4, pos, oldest); };
    float f[2];
    cap_and_mask<LARGE_CAP>(a, s, sc, row_factor, masked, seen, f);
    Weights w;
    w.begin(sc, mc);
    f32x16 after = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      after = Fp16::mfma32(kf[ks], qf[ks], after);
#pragma unroll
      for (int i = ks * 16 / KS; i < (ks + 1) * 16 / KS; ++i) w.take(s, f, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    read_v(0);
    settle(w, s, f, sc, m, mc, l, o);
    const u32x4 pf[2] = {w.packed(0), w.packed(1)};
    read_v(1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        o[d] = Fp16::mfma32(vf[h][d], pf[h], o[d]);
#pragma unroll
        for (int u = (h * DT + d) * kHalf / DT; u < (h * DT + d + 1) * kHalf / DT; ++u) decode_unit(n, u, stage ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    load(tile + 2, n);
    s = after;
  };

  // ---- main loop: tile j from stage j % 2; tile j + 1 is decoded into the other one and j + 2 requested under it ----
  load(0, 0);
  load(0, 1);
  {  // rows of q to the lanes that multiply them, by way of the second stage
    static_assert(WR * 32 * P <= kStage, "the rows fit a stage");
    const unsigned rows = lds0 + unsigned(kStage + wr * 32 * P);
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
  row_factor = (a.bf16 ? row_to_fp16<Bf16>(qf, a.negate != 0) : row_to_fp16<Fp16>(qf, a.negate != 0)) * C::kUnit;
  store_scales(0);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int u = 0; u < 2 * kHalf; ++u) decode_unit(n, u, 0);
    load(1, n);
  }
  if constexpr (WD == 1) {
    stage_barrier();
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s = Fp16::mfma32(*reinterpret_cast<const lds_v4*>(size_t(k_rd ^ unsigned(ks * 32))), qf[ks], s);
    for (int j = 0; j < tiles; ++j) {
      step(j, std::integral_constant<int, 0>{}, s);
      stage_barrier();
      step(j, std::integral_constant<int, 1>{}, s);
      stage_barrier();
    }
  } else {
    for (int j = 0; j < tiles; ++j) {
      stage_barrier();
      pair_tile(j, j & 1);
    }
  }
  l = swap_add(l);
  if constexpr (WD == 2) {  // the waves' parts of the sum
    const unsigned sums = lds0 + unsigned(kTops + (lane & 31) * 4);
    stage_barrier();
    *reinterpret_cast<lds_float*>(size_t(sums + unsigned(wave * 128))) = l;
    stage_barrier();
    l += *reinterpret_cast<const lds_float*>(size_t(sums + unsigned((wave ^ WR) * 128)));
  }

  // ---- rows to out, or to the parts that are joined: through LDS, so that a store covers whole lines of a row ----
  // where the lane's rows go, worked out again here: kept from above it would cost registers in the loop
  int row_first = t.row0;
  asm volatile("" : "+s"(row_first));
  __syncthreads();  // the stages are free
  constexpr int kRowB = DT * 64, kPad = kRowB + 16, kPadF = 128 + 16;  // a wave's part of a row; 32 FP32 values of one
  const unsigned mine_rows = lds0 + unsigned(wave * 32 * kPad);
  const int rl = lane & 31;
  const bool there = wr * 32 + rl < t.rows;
  const int row_at = min(row_first + wr * 32 + rl, last_row), token_at = row_at / a.group;
  const int token = t.seq.first + token_at, head = kvh * a.group + (row_at - token_at * a.group);
  const bool parts = range.splits > 1;
  const long long to = !there  ? -1
                       : parts ? (((long long)token * a.q_heads + head) * a.splits + z) * (D + 4) + wd * DT * 32
                               : token * a.o_stride + head * D + wd * DT * 32;
  const unsigned row = mine_rows + unsigned(rl * (parts ? kPadF : kPad));
  if (half == 0) *reinterpret_cast<lds_ll*>(size_t(row + unsigned(parts ? 128 : kRowB))) = to;
  // decode8's order undone
  const auto four = [&](int d, int i) { return f32x4{o[d][4 * i], o[d][4 * i + 2], o[d][4 * i + 1], o[d][4 * i + 3]}; };
  if (parts) {
    if (there && half == 0 && wd == 0) {
      a.part[to + D] = m == -INFINITY ? -INFINITY : mc;
      a.part[to + D + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<lds_f4*>(size_t(row + unsigned((8 * i + 4 * half) * 4))) = four(d, i) * C::kUnit;
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
    const float inv = l == 0.f ? 0.f : C::kUnit / l;
    const auto rows_as = [&](auto type) {
      using E = decltype(type);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 v = four(d, i);
          if (l == 0.f) v = f32x4{};  // nothing seen
          v *= inv;
          *reinterpret_cast<lds_v2*>(size_t(row + unsigned((32 * d + 8 * i + 4 * half) * 2))) =
              u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
        }
    };
    if (a.bf16)
      rows_as(Bf16{});
    else
      rows_as(Fp16{});
    __builtin_amdgcn_s_waitcnt(0xc07f);
    constexpr int kOutPieces = kRowB / 16;
#pragma unroll
    for (int j = 0; j < kOutPieces / 2; ++j) {
      const int piece = j * 64 + lane, from_row = piece / kOutPieces, c = piece % kOutPieces;
      const unsigned from = mine_rows + unsigned(from_row * kPad);
      const long long at = *reinterpret_cast<const lds_ll*>(size_t(from + unsigned(kRowB)));
      const u32x4 v = *reinterpret_cast<const lds_v4*>(size_t(from + unsigned(c * 16)));
      if (at >= 0) store_16_bytes(a.out + at + c * 8, v);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
}

template <typename C, int D, bool LARGE_CAP>
int launch(const Kv8Args& a, const Shape& s, hipStream_t stream) {
  if (!fits_launch(a, s)) return GIE_HIP_EUNSUPPORTED;
  const int grid = int((long long)s.slots * s.splits * a.kv_heads);
  int rc;
  if (s.wide) {
    constexpr int WD = D == 256 ? 2 : 1, WR = kWideRows / 32;
    constexpr int exchange = WD == 1 ? 0 : WR * WD * (2048 + 4 + 128);
    constexpr int bytes = 2 * 2 * kWideKeys * kPitch<D> + 2 * WR * 16 + exchange, rows = WR * WD * 32 * (D / WD * 2 + 16);
    static_assert(rows <= bytes && WR * WD * 32 * 144 <= bytes, "rows on their way out fit the stages");
    rc = start(wide_kernel<C, D, WD, LARGE_CAP>, grid, 256 * WD, bytes, stream, a);
  } else {
    constexpr int WK = D == 256 ? 4 : 8, NST = 2;
    constexpr int bytes = WK * NST * 2 * kNarrowKeys * kPitch8<D>, join = WK * 256 + WK * 32 * (D + 4) * 4;
    rc = start(narrow_kernel<C, D, WK, NST, LARGE_CAP>, grid, 64 * WK, bytes > join ? bytes : join, stream, a);
  }
  if (rc != GIE_HIP_OK || s.splits == 1) return rc;
  return a.bf16 ? join_parts<Bf16, D>(a, s, stream) : join_parts<Fp16, D>(a, s, stream);
}

template <typename C, bool LARGE_CAP>
int launch(const Kv8Args& a, const Shape& s, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch<C, 64, LARGE_CAP>(a, s, stream);
    case 96: return launch<C, 96, LARGE_CAP>(a, s, stream);
    case 128: return launch<C, 128, LARGE_CAP>(a, s, stream);
    default: return launch<C, 256, LARGE_CAP>(a, s, stream);
  }
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_kv8_attention_workspace(const gie_kv_geom* g) {
  if (!valid_paged(g) || g->total_tokens == 0) return 0;
  return parts_bytes(*g, shape_of(*g));
}

extern "C" int gie_hip_kv8_attention(int dtype, int code, const gie_kv_geom* g, const void* q, const void* k_pages,
                                     const void* v_pages, const float* k_scales, const float* v_scales,
                                     const int* q_starts, const int* seq_lens, const int* page_table, void* out,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_paged(g) || !valid_code(code)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  // (a scale of 0 times a masked score is a NaN)
  if (!std::isfinite(g->scale) || g->scale == 0 || !std::isfinite(g->softcap)) return GIE_HIP_EINVAL;
  if ((long long)g->kv_heads * (g->page_size / 16) > 0x7fffffff / g->num_pages) return GIE_HIP_EUNSUPPORTED;  // blocks
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_attention(g, q, k_pages, v_pages, q_starts, seq_lens, page_table, out)) return GIE_HIP_EINVAL;
  if (!k_scales || !v_scales || k_scales == v_scales || !aligned_to(k_scales, 4) || !aligned_to(v_scales, 4))
    return GIE_HIP_EINVAL;
  const Shape shape = shape_of(*g);
  const size_t need = parts_bytes(*g, shape);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return GIE_HIP_EINVAL;
  Kv8Args a{};
  a.k_pages = static_cast<const uint8_t*>(k_pages);
  a.v_pages = static_cast<const uint8_t*>(v_pages);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.page_blocks = unsigned(g->kv_heads) * unsigned(g->page_size / 16);
  a.bf16 = dtype == GIE_HIP_BF16;
  const bool large_cap = fill_args(a, g, shape, q, q_starts, seq_lens, page_table, out, workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = g->head_dim;
  if (code == GIE_HIP_KV_INT8)
    return large_cap ? launch<Int8Code, true>(a, shape, D, s) : launch<Int8Code, false>(a, shape, D, s);
  return large_cap ? launch<E4m3Code, true>(a, shape, D, s) : launch<E4m3Code, false>(a, shape, D, s);
}
