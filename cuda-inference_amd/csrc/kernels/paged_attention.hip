// Attention of new tokens over a paged key/value cache:
//   out[t][h] = sum_j softmax_j(s_j) v_j,  s_j = scale * q[t][h] . k_j  (or softcap * tanh(that / softcap)),
// over the positions j <= p (and j > p - window or j < sinks) of the token's sequence, in one pass over the keys with the
// running maximum m and sum l of the softmax.
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
#include "attention_common.h"

namespace gie_hip {
namespace {

struct PagedArgs : AttnArgs {
  const uint16_t* k_pages;
  const uint16_t* v_pages;
};

// WD waves take the same rows and a part of the head's values each: they work out the same scores (the first product is
// theirs in full) and sum their part of V. LARGE_CAP: scores under a cap past kExpCap.
template <typename E, int D, int WR, int WK, int WD, int NST, bool LARGE_CAP>
__global__ __launch_bounds__(64 * WR * WK * WD, WK == 2 ? 1 : 2) void attention_kernel(PagedArgs a) {
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
  const int tiles = min(range.per_split, range.tiles - tile_first);  // of the workgroup; this wave: wk, wk + WK, ...
  // first position of a tile of the workgroup
  const int turn = range.sink_tiles - tile_first, sink0 = tile_first * TT;
  const int key0 = sink0 + range.lo - range.sink_tiles * TT;
  const auto key_of = [&](int tile) { return tile * TT + (tile < turn ? sink0 : key0); };

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
      const int gran = min((key_of(tile) >> 4) + (WR > 1 ? wr : g), (a.capacity >> 4) - 1);
      const int pg = div_magic(gran, a.page_magic, a.page_shift);
      page[g] = table[__builtin_amdgcn_readfirstlane(pg)];
      slot16[g] = gran - pg * a.page16;
    }
  };
  const auto issue = [&](int tile, int stage) {
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const int gi = WR > 1 ? wr : g;
      const int at = key_of(tile) + gi * 16;
      const bool there = page[g] >= 0 && page[g] < a.num_pages && tile < tiles;
      const int bytes = there ? min(max(range.hi - at, 0), 16) * 2 * D : 0;
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
    const int at0 = key_of(tile), oldest = a.window > 0 ? pos - a.window : -1;
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
          const uint32_t seen = sees(a, key, pos, oldest) ? ~0u : 0u;
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
                o[d][4 * i + e] += __uint_as_float(value & seen);
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
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = at + 8 * (i / 4) + 4 * half + i % 4;
          s[i] = sees(a, key, pos, oldest) ? s[i] : -INFINITY;
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

template <typename E, int D, bool LARGE_CAP>
int launch(const PagedArgs& a, const Shape& s, hipStream_t stream) {
  if (!fits_launch(a, s)) return GIE_HIP_EUNSUPPORTED;
  const long long grid = (long long)s.slots * s.splits * a.kv_heads;
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
  return rc != GIE_HIP_OK || s.splits == 1 ? rc : join_parts<E, D>(a, s, stream);
}

template <typename E, bool LARGE_CAP>
int launch(const PagedArgs& a, const Shape& s, int head_dim, hipStream_t stream) {
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

extern "C" size_t gie_hip_kv_attention_workspace(const gie_kv_geom* g) {
  if (!valid_paged(g) || g->total_tokens == 0) return 0;
  return parts_bytes(*g, shape_of(*g));
}

extern "C" int gie_hip_kv_attention(int dtype, const gie_kv_geom* g, const void* q, const void* k_pages,
                                    const void* v_pages, const int* q_starts, const int* seq_lens,
                                    const int* page_table, void* out, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  // (a scale of 0 times a masked score is a NaN)
  if (!std::isfinite(g->scale) || g->scale == 0 || !std::isfinite(g->softcap)) return GIE_HIP_EINVAL;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_attention(g, q, k_pages, v_pages, q_starts, seq_lens, page_table, out)) return GIE_HIP_EINVAL;
  const size_t need = gie_hip_kv_attention_workspace(g);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return GIE_HIP_EINVAL;
  const Shape shape = shape_of(*g);
  PagedArgs a{};
  a.k_pages = static_cast<const uint16_t*>(k_pages);
  a.v_pages = static_cast<const uint16_t*>(v_pages);
  const bool large_cap = fill_args(a, g, shape, q, q_starts, seq_lens, page_table, out, workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = g->head_dim;
  if (dtype == GIE_HIP_FP16) return large_cap ? launch<Fp16, true>(a, shape, D, s) : launch<Fp16, false>(a, shape, D, s);
  return large_cap ? launch<Bf16, true>(a, shape, D, s) : launch<Bf16, false>(a, shape, D, s);
}

extern "C" size_t gie_hip_paged_attention_workspace(const gie_paged_geom* g) {
  if (!g) return 0;
  const gie_kv_geom geom = widened(*g);
  return gie_hip_kv_attention_workspace(&geom);
}

extern "C" int gie_hip_paged_attention(int dtype, const gie_paged_geom* g, const void* q, const void* k_pages,
                                       const void* v_pages, const int* q_starts, const int* seq_lens,
                                       const int* page_table, void* out, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (!g) return GIE_HIP_EINVAL;
  const gie_kv_geom geom = widened(*g);
  return gie_hip_kv_attention(dtype, &geom, q, k_pages, v_pages, q_starts, seq_lens, page_table, out, workspace,
                              workspace_bytes, stream);
}
