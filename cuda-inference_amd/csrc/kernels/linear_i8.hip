// Matrix product in 8-bit integers with scales for each token and output channel:
//   y[t][n] = round(relu?(float(sum_k q[t][k] w[n][k]) * (x_scale[t] * w_scale[n]) + bias[n]))
// The sum runs on the i8 matrix cores into int32 (exact in any order); scales, bias and the one rounding in FP32.
//
// Two forms, by the number of tokens:
//   * few tokens (<= 16): the weights' one pass through memory is all there is. A workgroup owns 16 output channels and
//     its 8 waves take every 8th step of 64 input values of them, straight from memory into the operands of
//     16x16x64 MFMAs, 8 steps in flight (64 KiB for a compute unit); their sums meet in LDS. Where x is not in 8 bits yet
//     and short (up to 4 tokens, 32 Ki values), every workgroup quantizes it for itself under the weights' loads: a
//     launch before this one costs 3.3 us. 1x4096x4096: 8.6 us, of which the 16.8 MB of weights are 3.6 at the copy's
//     rate; the rest is a launch, one chain x -> scale -> 8 bits -> product, and the moves of 211 scalars that do not fit
//     their registers (the form that reads x in 8 bits has none); 2x8192x8192 18 us, 3.7 TB/s.
//   * tiles of 32 to 256 tokens and channels: 128 input values of each in LDS at a time, NST stages of direct loads,
//     32x32x32 MFMAs. Channels are the rows of a product and tokens its columns, so a lane holds 4 neighbouring channels of
//     one token; the finished tile goes through LDS and out in whole rows. Rows of 128 bytes with their 16-byte chunks
//     permuted by the row meet no LDS bank twice. Tiles of 32 are shared by 4 waves along the input values. Where there
//     are too few tiles to fill the device they are split over parts of the input values: int32 partial sums in the
//     workspace and a second launch that joins them (integers: the order does not matter).
//     4096x4096x16384: 265-288 us with its quantization (11 us), 1.9-2.1 POP/s; 8192x8192x8192 in 8 bits already: 473-486
//     us, 2.3 POP/s (the library product of the same size 2.13). The matrix cores are busy half of the time; without
//     loads the same products take 218 us, loads alone 217: L2 -> LDS runs at 10-13 TB/s, whatever the number of stages
//     (2, 3, 4 measured), the order of a row's chunks (measured without the permutation) and the order of the tiles (1 to
//     16 of tokens in a run: 265-283 us). 64x8192x8192: 17 us for 67 MB of weights, 4.0 TB/s, and 4 us for the join.
// Rows that no 16-byte piece fits (ld or address) go through registers instead of direct loads, in pieces of any
// alignment, up to 4 slices ahead: 429x9468x1888 40 us against 36 at 9472.
#include "quantize_common.h"

#include "lds_pipe.h"

namespace gie_hip {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) u32x4 lds_v4;
typedef __attribute__((address_space(3))) f32x4 lds_f4;
typedef __attribute__((address_space(3))) float lds_f;

struct LinArgs {
  const int8_t* x;
  const float* x_scale;
  const int8_t* w;
  const float* w_scale;
  const void* bias;
  void* y;
  int* part;        // splits > 1: [split][tokens][out_features]
  const void* x16;  // few tokens: x before its quantization, or null
  long long ld_x, ld_w, ld_y;
  int M, N, K;
  int relu;
  int splits, per_split;  // parts of the input values, and their steps of 128
  int tiles_m, tiles_n;
  int y_vec;  // rows of y in 16-byte pieces (whole lines from LDS)
};

template <typename E>
constexpr int kBytesOf = 2;
template <>
constexpr int kBytesOf<F32> = 4;

// values k .. k + 15 of a row, zeros from K on; nothing behind the row's end is read
__device__ __forceinline__ u32x4 load16_upto(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return load_16_bytes(row + k);
  u32x4 v = {};
  for (int i = 0; i < 16; ++i)
    if (k + i < K) v[i / 4] |= uint32_t(uint8_t(row[k + i])) << (8 * (i % 4));
  return v;
}

__device__ __forceinline__ float finish(int acc, float scale, float w_scale, float bias, int relu) {
  float v = float(acc) * (scale * w_scale);  // the scales first: acc times a large one could pass FP32
  v += bias;
  return relu && v < 0.f ? 0.f : v;  // a NaN stays
}

template <typename E>
__device__ __forceinline__ float bias_at(const void* bias, int n) {
  return bias != nullptr ? load_value<E>(bias, n) : 0.f;
}

// ---------------------------------------------------------------------------------------------- tiles
// WK waves share a part of the tile and take every WK-th 32 of a stage's input values; NST stages
template <typename E, int BM, int BN, int WM, int WN, int WK, int NST, bool ALIGNED>
__global__ __launch_bounds__(64 * WM * WN * WK, 1) void tile_kernel(LinArgs a) {
  constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32x32 products of a wave
  constexpr int kRows = BM + BN, kStage = kRows * 128;
  constexpr int IPW = kRows / 8 / kWaves;  // loads of 8 rows for each wave
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = int(threadIdx.x), lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN);

  // tile: workgroup L runs on XCD L % 8, which takes a run of neighbouring tiles: 4 of tokens for each of channels, so
  // that those which run together share rows of x and w in its L2
  int tm, tn;
  {
    const int total = a.tiles_m * a.tiles_n;
    const int L = int(blockIdx.x), xcd = L & 7;
    const int lo = total / 8, more = total % 8;
    const int id = xcd * lo + min(xcd, more) + (L >> 3);
    const int group = 4 * a.tiles_n, first = id / group * 4, high = min(4, a.tiles_m - first);
    tm = first + id % group % high;
    tn = id % group / high;
  }
  const int m0 = tm * BM, n0 = tn * BN;
  const int k_first = int(blockIdx.y) * a.per_split * 128;
  const int k_last = min(a.K, k_first + a.per_split * 128);
  const int steps = (k_last - k_first + 127) / 128;

  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds));
  i32x16 acc[TN][TM] = {};

  // ---- loads: instruction i of the wave covers rows 8 (wave IPW + i) .. + 7 of the stage, x first ----
  const int r0 = lane >> 3;
  const int chunk_even = (lane & 7) ^ (r0 >> 1), chunk_odd = chunk_even ^ 4;
  const auto uniform = [](v4i r) {
    return v4i{__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y),
               __builtin_amdgcn_readfirstlane(r.z), __builtin_amdgcn_readfirstlane(r.w)};
  };
  const auto issue = [&](int step, int stage) {
    const int k0 = k_first + step * 128, left = k_last - k0;
    // bytes to the end of the last row, its last 16-byte piece whole (it holds a byte of the row, and a piece of 16 lies
    // in one page): the hardware would drop a word that passes the end
    const long long rx = (long long)(min(BM, a.M - m0) - 1) * a.ld_x + ((left + 15) & ~15);
    const long long rw = (long long)(min(BN, a.N - n0) - 1) * a.ld_w + ((left + 15) & ~15);
    v4i sx = uniform(make_vsharp(a.x + m0 * a.ld_x + k0, left > 0 ? int(rx) : 0));
    v4i sw = uniform(make_vsharp(a.w + n0 * a.ld_w + k0, left > 0 ? int(rw) : 0));
    // a vector instruction may have written these scalar registers: loads may read them 5 cycles later
    asm volatile("s_nop 4" : "+s"(sx), "+s"(sw));
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int at = wave * IPW + i;  // uniform
      const bool is_x = at < BM / 8;
      const int row = (is_x ? at : at - BM / 8) * 8 + r0;
      const int chunk = at & 1 ? chunk_odd : chunk_even;
      const int off = chunk * 16 < left ? row * int(is_x ? a.ld_x : a.ld_w) + chunk * 16 : kOut;
      if (is_x)
        dma16(sx, lds0 + unsigned(stage * kStage + at * 1024), off);
      else
        dma16(sw, lds0 + unsigned(stage * kStage + at * 1024), off);
    }
  };
  // rows of any alignment: 16 bytes for each thread and round through registers
  constexpr int kRounds = kRows * 8 / kThreads;
  constexpr int kAhead = kRounds <= 4 ? 4 : 1;  // slices held
  u32x4 held[ALIGNED ? 1 : kAhead][ALIGNED ? 1 : kRounds];
  const int8_t* rows[ALIGNED ? 1 : kRounds];  // of this thread's pieces; those past the last repeat it and are not stored
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int row = (i * kThreads + tid) >> 3;
      rows[i] = row < BM ? a.x + min(m0 + row, a.M - 1) * a.ld_x : a.w + min(n0 + row - BM, a.N - 1) * a.ld_w;
    }
  }
  const auto fetch = [&](int step, u32x4* to) {
    const int k0 = k_first + step * 128, k = k0 + (tid & 7) * 16;
    if (k0 + 128 <= k_last) {
#pragma unroll
      for (int i = 0; i < kRounds; ++i) to[i] = load_16_bytes(rows[i] + k);
    } else {
#pragma unroll
      for (int i = 0; i < kRounds; ++i) to[i] = k < k_last ? load16_upto(rows[i], k, k_last) : u32x4{};
    }
  };
  const auto put = [&](int stage, const u32x4* from) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int c = i * kThreads + tid, row = c >> 3, slot = (c & 7) ^ ((row >> 1) & 7);
      *reinterpret_cast<lds_v4*>(size_t(lds0 + unsigned(stage * kStage + row * 128 + slot * 16))) = from[i];
    }
  };

  // ---- fragments: lane row (lane & 31), 16 bytes at 32 ks + 16 half ----
  const unsigned swz = unsigned((half ^ ((lane >> 1) & 7)) << 4);
  const unsigned x_rd = lds0 + unsigned((wm * TM * 32 + (lane & 31)) * 128) + swz;
  const unsigned w_rd = lds0 + unsigned((BM + wn * TN * 32 + (lane & 31)) * 128) + swz;
  const auto compute = [&](int stage) {
    const unsigned so = unsigned(stage * kStage);
#pragma unroll
    for (int kk = 0; kk < 4 / WK; ++kk) {
      const int ks = kk * WK + wk;
      u32x4 xf[TM], wf[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
        xf[i] = *reinterpret_cast<const lds_v4*>(size_t(((x_rd + so) ^ unsigned(ks * 32)) + unsigned(i * 32 * 128)));
#pragma unroll
      for (int i = 0; i < TN; ++i)
        wf[i] = *reinterpret_cast<const lds_v4*>(size_t(((w_rd + so) ^ unsigned(ks * 32)) + unsigned(i * 32 * 128)));
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, wf[n]),
                                                            __builtin_bit_cast(i32x4, xf[m]), acc[n][m], 0, 0, 0);
    }
  };
  // a 16-byte chunk that the row ends in holds bytes of what lies behind it: they are cleared in x, so what w holds there
  // does not matter
  const auto clear_tail = [&](int stage) {
    const int left = (k_last - k_first) % 128, bytes = left % 16;
    if (bytes == 0) return;
    for (int row = tid; row < BM; row += kThreads) {
      const int slot = (left >> 4) ^ ((row >> 1) & 7);
      lds_v4* at = reinterpret_cast<lds_v4*>(size_t(lds0 + unsigned(stage * kStage + row * 128 + slot * 16)));
      u32x4 v = *at;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int keep = min(max(bytes - 4 * e, 0), 4);
        v[e] &= keep == 4 ? ~0u : (1u << (8 * keep)) - 1u;
      }
      *at = v;
    }
    stage_barrier();
  };

  if constexpr (ALIGNED) {
    // loads past the last slice read nothing, so that every wait counts the same
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(s, s);
    int stage = 0;
    for (int s = 0; s < steps; ++s) {
      wait_vm<(NST - 2) * IPW>();
      stage_barrier();
      issue(s + NST - 1, stage == 0 ? NST - 1 : stage - 1);
      if (s + 1 == steps) clear_tail(stage);
      compute(stage);
      stage = stage + 1 == NST ? 0 : stage + 1;
    }
    wait_vm<0>();
  } else {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(u, held[u]);
    for (int s = 0; s < steps; s += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u >= steps) break;
        put((s + u) & 1, held[u]);
        fetch(s + u + kAhead, held[u]);
        __syncthreads();
        compute((s + u) & 1);
      }
    }
  }
  __syncthreads();

  if constexpr (WK > 1) {  // the waves' sums meet in the first's
    static_assert(WM == 1 && WN == 1, "one part of the tile");
    lds_v4* sums = reinterpret_cast<lds_v4*>(size_t(lds0));
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (wk > 0)
            sums[(((wk - 1) * TN + n) * TM + m) * 256 + g * 64 + lane] =
                u32x4{uint32_t(acc[n][m][4 * g]), uint32_t(acc[n][m][4 * g + 1]), uint32_t(acc[n][m][4 * g + 2]),
                      uint32_t(acc[n][m][4 * g + 3])};
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int w = 0; w < WK - 1; ++w)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const u32x4 v = sums[((w * TN + n) * TM + m) * 256 + g * 64 + lane];
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[n][m][4 * g + e] += int(v[e]);
            }
    }
    __syncthreads();
  }

  // ---- 32 tokens at a time through the wave's own part of LDS, then out in rows ----
  if (a.splits > 1) {
    if (WK > 1 && wk > 0) return;
    int* part = a.part + (long long)blockIdx.y * a.M * a.N;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int t = m0 + (wm * TM + m) * 32 + (lane & 31);
      if (t >= a.M) continue;
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = n0 + (wn * TN + n) * 32 + 8 * g + 4 * half;
          int* dst = part + (long long)t * a.N + c;
          if (a.N % 4 == 0 && c < a.N) {
            *reinterpret_cast<i32x4*>(dst) =
                i32x4{acc[n][m][4 * g], acc[n][m][4 * g + 1], acc[n][m][4 * g + 2], acc[n][m][4 * g + 3]};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e < a.N) dst[e] = acc[n][m][4 * g + e];
          }
        }
    }
    return;
  }
  constexpr int kE = kBytesOf<E>, kRowB = TN * 32 * kE, kPad = kRowB + 16;
  const unsigned tile = lds0 + unsigned(wave * 32 * kPad);
  const unsigned scales = lds0 + unsigned(kWaves * 32 * kPad);  // of the tile's channels, and their biases behind them
  for (int c = tid; c < BN; c += kThreads) {
    const int n = min(n0 + c, a.N - 1);
    *reinterpret_cast<lds_f*>(size_t(scales + c * 4)) = a.w_scale[n];
    *reinterpret_cast<lds_f*>(size_t(scales + (BN + c) * 4)) = bias_at<E>(a.bias, n);
  }
  __syncthreads();
  if (WK > 1 && wk > 0) return;
  const int c0 = n0 + wn * TN * 32;  // the wave's first channel
  const unsigned mine = scales + unsigned((wn * TN * 32 + 4 * half) * 4);
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int t0 = m0 + (wm * TM + m) * 32;
    if (t0 >= a.M) break;
    const float xs = a.x_scale[min(t0 + (lane & 31), a.M - 1)];
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      asm volatile("" ::: "memory");  // a part's sums at a time: all of them at once would not fit the registers
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = n * 32 + 8 * g;
        const f32x4 ws = *reinterpret_cast<const lds_f4*>(size_t(mine + col * 4));
        const f32x4 bs = *reinterpret_cast<const lds_f4*>(size_t(mine + (BN + col) * 4));
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = finish(acc[n][m][4 * g + e], xs, ws[e], bs[e], a.relu);
        const unsigned at = tile + unsigned((lane & 31) * kPad + (col + 4 * half) * kE);
        if constexpr (kE == 4)
          *reinterpret_cast<lds_v4*>(size_t(at)) =
              u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        else
          *reinterpret_cast<__attribute__((address_space(3))) u32x2*>(size_t(at)) =
              u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // the wave's own writes
    constexpr int kLanesRow = kRowB / 16, kRowsIt = 64 / kLanesRow > 0 ? 64 / kLanesRow : 1;
    static_assert(kLanesRow <= 64, "a row fits one instruction");
#pragma unroll 4
    for (int r = 0; r < 32; r += kRowsIt) {
      const int row = r + lane / kLanesRow, piece = lane % kLanesRow;
      const int t = t0 + row, c = c0 + piece * (16 / kE);
      const u32x4 v = *reinterpret_cast<const lds_v4*>(size_t(tile + unsigned(row * kPad + piece * 16)));
      if (t >= a.M) continue;
      char* dst = static_cast<char*>(a.y) + (t * a.ld_y + c) * kE;
      if (a.y_vec && c + 16 / kE <= a.N) {
        *reinterpret_cast<u32x4*>(dst) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 16 / kE; ++e) {
          if (c + e >= a.N) break;
          if constexpr (kE == 4)
            reinterpret_cast<uint32_t*>(dst)[e] = v[e];
          else
            reinterpret_cast<uint16_t*>(dst)[e] = uint16_t(v[e / 2] >> (16 * (e & 1)));
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
}

// ---------------------------------------------------------------------------------------------- join
template <typename E>
__global__ __launch_bounds__(256) void join_kernel(LinArgs a) {
  const long long total = (long long)a.M * a.N, pieces = (total + 3) / 4;
  for (long long p = (long long)blockIdx.x * 256 + threadIdx.x; p < pieces; p += (long long)gridDim.x * 256) {
    const long long i = p * 4;
    const bool whole = a.N % 4 == 0;
    int acc[4] = {};
    for (int z = 0; z < a.splits; ++z) {
      const int* src = a.part + z * total + i;
      if (whole) {
        const i32x4 v = *reinterpret_cast<const i32x4*>(src);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < total) acc[e] += src[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e >= total) break;
      const long long t = (i + e) / a.N;
      const int n = int((i + e) - t * a.N);
      store_value<E>(a.y, t * a.ld_y + n,
                     finish(acc[e], a.x_scale[t], a.w_scale[n], bias_at<E>(a.bias, n), a.relu));
    }
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
constexpr int kFew = 16, kFewWaves = 8, kFewThreads = 64 * kFewWaves;

// FUSED: x16 is quantized here, into LDS; otherwise x is read as the weights are
template <typename E, bool FUSED>
__global__ __launch_bounds__(kFewThreads) void few_kernel(LinArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ i32x4 sums[kFewWaves][64];
  __shared__ float scales[kFew];
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = int(blockIdx.x) * 16;
  const int row = lane & 15, part = (lane >> 4) * 16;
  const int K16 = (a.K + 15) & ~15;
  const int8_t* w = a.w + min(n0 + row, a.N - 1) * a.ld_w;
  const int token = min(row, a.M - 1);
  const int8_t* x = FUSED ? reinterpret_cast<const int8_t*>(lds) + token * K16 : a.x + token * a.ld_x;
  const int steps = (a.K + 63) / 64;
  constexpr int U = 8;  // steps in flight
  u32x4 wf[U];
  const auto load_w = [&](int s) {
    const int k = s * 64 + part;
    return s < steps && k < a.K ? load16_upto(w, k, a.K) : u32x4{};
  };
  if constexpr (FUSED) {
    // x first: its way to 8 bits is the longer one, and the weights arrive under it
    constexpr int kPer = 16 / kBytesOf<E>, kKeep = 4;
    for (int t = 0; t < a.M; ++t) {
      const char* row = static_cast<const char*>(a.x16) + t * a.ld_x * kBytesOf<E>;
      const int pieces = a.K / kPer;
      u32x4 keep[kKeep];
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        const int p = i * kFewThreads + tid;
        keep[i] = p < pieces ? load_16_bytes(row + p * 16ll) : u32x4{};
      }
      if (t == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) wf[u] = load_w(wave + u * kFewWaves);
      }
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        float f[8];
        unpack<E>(keep[i], f);
#pragma unroll
        for (int e = 0; e < kPer; ++e) most = magnitude_max(most, f[e]);
      }
      const int rest = min(pieces, kKeep * kFewThreads) * kPer;  // value by value from here
      for (int k = rest + tid; k < a.K; k += kFewThreads) most = magnitude_max(most, load_value<E>(a.x16, t * a.ld_x + k));
      most = block_magnitude_max<kFewThreads>(most);
      const RowScale s = row_scale(most);
      if (tid == 0) scales[t] = s.scale;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        const int p = i * kFewThreads + tid;
        if (p < pieces) quantize_piece<E>(keep[i], s.inverse, lds + t * K16 + p * kPer);
      }
      for (int k = rest + tid; k < K16; k += kFewThreads)
        lds[t * K16 + k] = k < a.K ? uint8_t(quantize_value(load_value<E>(a.x16, t * a.ld_x + k), s.inverse)) : 0;
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) wf[u] = load_w(wave + u * kFewWaves);
  }
  i32x4 acc = {};
  for (int s0 = wave; s0 < steps; s0 += U * kFewWaves) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * kFewWaves;
      if (s >= steps) break;
      const int k = s * 64 + part;
      u32x4 xf = {};
      if (k < a.K) {
        if constexpr (FUSED)
          xf = *reinterpret_cast<const u32x4*>(x + k);
        else
          xf = load16_upto(x, k, a.K);
      }
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wf[u]), __builtin_bit_cast(i32x4, xf), acc, 0,
                                                  0, 0);
      wf[u] = load_w(s + U * kFewWaves);
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (tid < 64) {
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) acc += sums[v][lane];
    if (row < a.M) {
      const float xs = FUSED ? scales[row] : a.x_scale[row];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + (lane >> 4) * 4 + e;
        if (n < a.N)
          store_value<E>(a.y, row * a.ld_y + n, finish(acc[e], xs, a.w_scale[n], bias_at<E>(a.bias, n), a.relu));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
size_t round16(size_t n) { return (n + 15) / 16 * 16; }

bool valid(int dtype, const gie_linear_geom* g) {
  return g && (dtype == GIE_HIP_FP32 || dtype == GIE_HIP_FP16 || dtype == GIE_HIP_BF16) && g->tokens >= 0 &&
         g->in_features > 0 && g->in_features <= 131071 && g->out_features > 0 && g->ld_x >= g->in_features &&
         g->ld_w >= g->in_features && g->ld_y >= g->out_features;
}

enum Form { kFewForm, kTile32, kTile64, kTile128, kTile256 };
struct Plan {
  Form form;
  int tile, tiles_m, tiles_n, splits, per_split;  // tile: tokens and channels of one
};

// Square tiles of 256, 128, 64 and 32 tokens and channels. A larger one moves less from the L2 for each product, a smaller
// one leaves less of the device without work; times of a step (128 input values) as measured with 4096 of them: 2.1 us
// for a round of 256 tiles of 256; 0.85 us for up to 256 tiles of 128, 1.26 us for 512 of them (two to a compute unit);
// 0.33 us for up to 256 tiles of 64 and 0.27 us for each 256 more. Measured / so estimated, us: 4096x4096 70 / 67 (256),
// 84 / 81 (128), 144 / 138 (64); 1024x4096 55 / 67, 29.6 / 27, 42 / 35; 512x4096 - , 27 / 27, 19.6 / 17.
// With less than 192 tiles of 64, these and tiles of 32, whole or over parts of the input values, are weighed by what
// they move: L2 to LDS 14 TB/s (64) and 11.6 TB/s (32), weights 4.2 TB/s, less where the device is not full; 2.5 us and
// 4 TB/s for parts that are joined. Measured / so estimated, us: 64x4096x4096 10.9 (32, whole) 12.2 (64, 4 parts) / 5.8,
// 8.5; 64x8192x8192 22.0 (64, 2 parts) 25.3 (32) / 20, 23; 256x1024x16384 19.8 (64, 4 parts) 25.7 (32) / 14, 23, each
// without the 5 us that a call costs in any form.
Plan plan_of(const gie_linear_geom& g) {
  Plan p{};
  const long long M = g.tokens, N = g.out_features;
  const int steps = (g.in_features + 127) / 128;
  p.splits = 1;
  p.per_split = steps;
  if (M <= kFew) {
    p.form = kFewForm;
    return p;
  }
  const auto count = [&](int tile) { return (long long)((M + tile - 1) / tile) * ((N + tile - 1) / tile); };
  const auto rounds = [](long long n, int of) { return double((n + of - 1) / of); };
  if (count(64) >= 192) {
    const double us256 = 2.1 * rounds(count(256), 256);
    const double us128 = count(128) <= 256 ? 0.85 : 1.26 * rounds(count(128), 512);
    const double us64 = count(64) <= 256 ? 0.33 : 0.27 * rounds(count(64), 256);
    if (us256 <= us128 && us256 <= us64)
      p.form = kTile256, p.tile = 256;
    else if (us128 <= us64)
      p.form = kTile128, p.tile = 128;
    else
      p.form = kTile64, p.tile = 64;
  } else {
    double best = 0;
    for (int tile = 64; tile >= 32; tile /= 2) {
      for (int n = 1; n <= 16 && (n == 1 || steps / n >= 2); n *= 2) {
        const double full = count(tile) * n < 256 ? 256.0 / (count(tile) * n) : 1.0;
        const double l2 = count(tile) * 2.0 * tile * g.in_features / (tile == 64 ? 14e6 : 11.6e6);
        const double hbm = double(N) * g.in_features / 4.2e6;
        const double join = n == 1 ? 0 : 2.5 + 8.0 * M * N * n / 4e6;
        const double us = (l2 > hbm ? l2 : hbm) * full + join;
        if (p.tile == 0 || us < best) {
          best = us;
          p.form = tile == 64 ? kTile64 : kTile32, p.tile = tile;
          p.per_split = (steps + n - 1) / n;
        }
      }
    }
    p.splits = (steps + p.per_split - 1) / p.per_split;
  }
  p.tiles_m = int((M + p.tile - 1) / p.tile);
  p.tiles_n = int((N + p.tile - 1) / p.tile);
  return p;
}

// Quantized inside the product: one launch less, but every workgroup does it. us in one launch / in two, 16 bits: 1x4096x4096
// 7.8 / 9.4, 1x16384x4096 19.2 / 27.8, 1x28672x4096 31.4 / 48.2, 1x32768x8192 67.7 / 69.6, 4x8192x4096 14.7 / 14.9,
// 4x8192x8192 21.9 / 19.8; 32 bits: 1x14336x4096 18.8 / 27.8, 2x14336x8192 31.5 / 32.6. (Rows past what the threads keep
// are read a second time, value by value; that, too, is less than the second launch.)
bool fuses(const gie_linear_geom& g) { return g.tokens <= 4 && (long long)g.tokens * g.in_features <= 32 * 1024; }

template <typename E, int BM, int BN, int WM, int WN, int WK, int NST>
int run_tiles(const LinArgs& a, bool aligned, hipStream_t s) {
  constexpr int kStages = NST * (BM + BN) * 128;
  constexpr int kOutB = WM * WN * WK * 32 * (BN / WN * kBytesOf<E> + 16) + BN * 8;
  constexpr int kSums = (WK - 1) * BM * BN * 4;
  constexpr int most = kStages > kOutB ? kStages : kOutB, bytes = most > kSums ? most : kSums;
  auto kernel = tile_kernel<E, BM, BN, WM, WN, WK, NST, true>;
  if constexpr (BM < 256)
    if (!aligned) kernel = tile_kernel<E, BM, BN, WM, WN, WK, NST, false>;
  const int rc = set_lds_limit(reinterpret_cast<const void*>(kernel), bytes);
  if (rc != GIE_HIP_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3(unsigned(a.tiles_m * a.tiles_n), unsigned(a.splits)), dim3(64 * WM * WN * WK), bytes,
                     s, a);
  return GIE_HIP_OK;
}

template <typename E>
int run(const Plan& p, const LinArgs& a, bool aligned, hipStream_t s) {
  int rc = GIE_HIP_OK;
  switch (p.form) {
    case kFewForm: {
      const int bytes = a.x16 ? a.M * int(round16(a.K)) : 0;
      const dim3 grid((a.N + 15) / 16);
      if (a.x16)
        hipLaunchKernelGGL((few_kernel<E, true>), grid, dim3(kFewThreads), bytes, s, a);
      else
        hipLaunchKernelGGL((few_kernel<E, false>), grid, dim3(kFewThreads), 0, s, a);
      break;
    }
    case kTile32: rc = run_tiles<E, 32, 32, 1, 1, 4, 8>(a, aligned, s); break;
    case kTile64: rc = run_tiles<E, 64, 64, 2, 2, 1, 4>(a, aligned, s); break;
    case kTile128: rc = run_tiles<E, 128, 128, 2, 2, 1, 2>(a, aligned, s); break;
    case kTile256:
      rc = aligned ? run_tiles<E, 256, 256, 2, 4, 1, 2>(a, true, s) : run_tiles<E, 128, 128, 2, 2, 1, 2>(a, false, s);
      break;
  }
  if (rc != GIE_HIP_OK) return rc;
  if (a.splits > 1) {
    const long long pieces = ((long long)a.M * a.N + 3) / 4;
    const long long blocks = (pieces + 255) / 256;
    hipLaunchKernelGGL(join_kernel<E>, dim3(unsigned(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_linear_i8_workspace(int dtype, const gie_linear_geom* g, int quantized) {
  if (!valid(dtype, g) || g->tokens == 0) return 0;
  const Plan p = plan_of(*g);
  size_t n = p.splits > 1 ? round16(size_t(p.splits) * g->tokens * g->out_features * 4) : 0;
  if (!quantized && !(p.form == kFewForm && fuses(*g)))
    n += round16(size_t(g->tokens) * round16(g->in_features)) + round16(size_t(g->tokens) * 4);
  return n;
}

extern "C" int gie_hip_linear_i8(int dtype, const gie_linear_geom* g, const void* x, const float* x_scale,
                                 const int8_t* w, const float* w_scale, const void* bias, void* y, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!valid(dtype, g)) return GIE_HIP_EINVAL;
  if (g->tokens == 0) return GIE_HIP_OK;
  if (!x || !w || !w_scale || !y || x == y) return GIE_HIP_EINVAL;
  const size_t esz = dtype == GIE_HIP_FP32 ? 4 : 2;
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if (at(y) % esz != 0 || at(bias) % esz != 0 || at(w_scale) % 4 != 0 || at(x_scale) % 4 != 0 ||
      (x_scale == nullptr && at(x) % esz != 0))
    return GIE_HIP_EINVAL;
  const size_t need = gie_hip_linear_i8_workspace(dtype, g, x_scale != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need || at(workspace) % 16 != 0)) return GIE_HIP_EINVAL;
  const Plan p = plan_of(*g);
  const bool own_x = x_scale == nullptr && !(p.form == kFewForm && fuses(*g));  // quantized into the workspace
  const long long ld_x = own_x ? (long long)round16(g->in_features) : g->ld_x;
  // direct loads into LDS take 16-byte pieces, and reach a tile's last row with a 32-bit offset
  const bool aligned = ld_x % 16 == 0 && g->ld_w % 16 == 0 && (own_x || at(x) % 16 == 0) && at(w) % 16 == 0 &&
                       ld_x < (1 << 22) && g->ld_w < (1 << 22);
  LinArgs a{};
  if (p.form == kFewForm) {
    if (g->out_features > (1 << 26)) return GIE_HIP_EUNSUPPORTED;
  } else {
    const int tile = p.form == kTile256 && !aligned ? 128 : p.tile;
    const long long tm = (g->tokens + (long long)tile - 1) / tile, tn = (g->out_features + (long long)tile - 1) / tile;
    if (tm * tn >= (1 << 23)) return GIE_HIP_EUNSUPPORTED;  // 512 threads for each: a launch's limit
    a.tiles_m = int(tm);
    a.tiles_n = int(tn);
  }
  a.x = static_cast<const int8_t*>(x);
  a.x_scale = x_scale;
  a.w = w;
  a.w_scale = w_scale;
  a.bias = bias;
  a.y = y;
  a.ld_x = ld_x;
  a.ld_w = g->ld_w;
  a.ld_y = g->ld_y;
  a.M = g->tokens;
  a.N = g->out_features;
  a.K = g->in_features;
  a.relu = g->relu ? 1 : 0;
  a.splits = p.splits;
  a.per_split = p.per_split;
  char* ws = static_cast<char*>(workspace);
  if (p.splits > 1) {
    a.part = reinterpret_cast<int*>(ws);
    ws += round16(size_t(p.splits) * g->tokens * g->out_features * 4);
  }
  if (own_x) {
    int8_t* q = reinterpret_cast<int8_t*>(ws);
    float* scale = reinterpret_cast<float*>(ws + round16(size_t(g->tokens) * ld_x));
    const int rc = gie_hip_quantize_rows(dtype, x, g->ld_x, g->tokens, g->in_features, q, ld_x, scale, stream);
    if (rc != GIE_HIP_OK) return rc;
    a.x = q;
    a.x_scale = scale;
  } else if (x_scale == nullptr) {
    a.x16 = x;
  }
  a.y_vec = g->ld_y * esz % 16 == 0 && at(y) % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GIE_HIP_FP32) return run<F32>(p, a, aligned, s);
  if (dtype == GIE_HIP_FP16) return run<Fp16>(p, a, aligned, s);
  return run<Bf16>(p, a, aligned, s);
}
