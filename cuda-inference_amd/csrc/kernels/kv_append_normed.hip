// Appends the keys and values of new tokens to a paged cache as kv_append does, with a norm of each head of q and k ahead
// of the rotation, into pages of the tokens' own type or into 8-bit pages with a scale for each block of 16 positions:
//   x'_d = x_d / sqrt(mean_d x_d^2 + eps) * w_d;  pairs (u, v) -> (u cos - v sin, u sin + v cos);  FP32 up to one rounding.
//
// Bytes-bound. A lane takes 16 values of a head, 8 pairs where they rotate, in 16-byte pieces; 4, 8 or 16 lanes make a
// head and sum its squares among them; the norms' weights lie in LDS (in registers they cost a third of the waves).
// Rows (q, and k and v of a cache in the tokens' type) go by token: a workgroup finds the places of one or more tokens and
// spreads all their heads over its lanes. Blocks of 8-bit pages go by position: a wave has one head's whole block, up to
// 16 tokens, in registers, so that the scale is the largest of them and every code is written once. Both parts are
// workgroups of one launch.
// A rotating part that is no multiple of 16 does not fall into such pieces: there a lane has 16 values side by side and
// finds the other one of a pair through LDS. That form takes 109 to 117 registers where the others take 56 to 73 up to
// head_dim 128 (half the waves), and its few rotating lanes go value by value while the others wait.
//
// 8192 tokens of 32 + 2 x 8 heads of 128, both norms: 33 us alone, 43 among calls on other data (206 MB, 4.8 TB/s; a large
// copy 4.7), with the weights in registers 54; into 8-bit pages 44 among calls on other data. With 6 of 128 values rotating
// 87 and 66. 64 tokens of one sequence each 4.1 us, into 8-bit pages 5.8 (the older codes of the blocks and their scales come
// on top of the chain lengths -> page -> store).
// 6089 tokens of 12 + 2 x 12 heads of 96 into 8-bit pages 20 us, 3.5 TB/s: two of eight lanes are idle, and every workgroup
// looks its block up, stages the weights and passes a barrier for four heads' 16 rows.
#include <cmath>
#include <type_traits>

#include "kv8_common.h"

namespace gie_hip {
namespace {

struct NormedArgs {
  gie_kv_geom g;
  const uint16_t* q;  // null: only keys and values
  const uint16_t* k;
  const uint16_t* v;
  const float* q_norm;  // null: not normed
  const float* k_norm;
  const float* cos;
  const float* sin;
  const int* q_starts;
  const int* seq_lens;
  const int* page_table;
  uint16_t* q_out;
  void* k_pages;
  void* v_pages;
  float* k_scales;
  float* v_scales;
};

// ---- 16 values a lane
template <int D>
constexpr int kHeadLanes = D == 64 ? 4 : D == 256 ? 16 : 8;  // of a head (6 of 8 at 96)

// how a head rotates: pairs of its halves or neighbours, in pieces of 16 values; kAny: either, any even number of values
enum Form { kHalves, kNeighbours, kAny };

// where a lane's 16 values lie in its head: 8 from `at`, 8 from `next`; pairs: they rotate (values i and 8 + i, or
// neighbours 2 i and 2 i + 1, by the angles from `angle` on; kAny: some of them do)
struct Unit {
  int at, next, angle;
  bool there, pairs;
};
template <Form F, int D>
__device__ __forceinline__ Unit unit_of(int unit, int rotary) {
  Unit u;
  u.there = unit < D / 16;
  u.pairs = u.there && unit * 16 < rotary;
  u.angle = unit * 8;
  u.at = u.pairs && F == kHalves ? unit * 8 : unit * 16;
  u.next = u.pairs && F == kHalves ? u.at + rotary / 2 : u.at + 8;
  return u;
}

template <typename E>
__device__ __forceinline__ void load_unit(const uint16_t* head, const Unit& u, float (&x)[16]) {
  const u32x4 a = u.there ? load_16_bytes(head + u.at) : u32x4{}, b = u.there ? load_16_bytes(head + u.next) : u32x4{};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = E::to_f32(uint16_t(a[i])), x[2 * i + 1] = E::to_f32(uint16_t(a[i] >> 16));
    x[8 + 2 * i] = E::to_f32(uint16_t(b[i])), x[9 + 2 * i] = E::to_f32(uint16_t(b[i] >> 16));
  }
}
// w: the weights in LDS (kept in registers they cost a third of the waves)
template <int D>
__device__ __forceinline__ void norm_unit(float (&x)[16], const float* w, const Unit& u, float eps) {
  float sum[2] = {};
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i % 2] = __builtin_fmaf(x[i], x[i], sum[i % 2]);
  float all = sum[0] + sum[1];
#pragma unroll
  for (int d = 1; d < kHeadLanes<D>; d <<= 1) all += __shfl_xor(all, d);
  // (off by an ulp: less than the sum)
  const float inv = __builtin_amdgcn_rsqf(all * (1.f / D) + eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(w + (u.there ? (i < 2 ? u.at : u.next - 8) + 4 * i : 0));
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = x[4 * i + e] * inv * v[e];
  }
}
// the weights of q's and k's norms, ones without one
template <int D>
__device__ __forceinline__ void stage_weights(const NormedArgs& a, float (*w)[D]) {
  for (int i = int(threadIdx.x); i < 2 * D; i += int(blockDim.x)) {
    const float* from = i < D ? a.q_norm : a.k_norm;
    w[i / D][i % D] = from ? from[i % D] : 1.f;
  }
}
// cos, sin: the position's rows of the tables; row: LDS for the head's values (kAny)
template <Form F>
__device__ __forceinline__ void turn_unit(float (&x)[16], const Unit& u, const gie_kv_geom& g, const float* cos,
                                          const float* sin, float* row) {
  const int half = g.rotary_dim / 2;
  if constexpr (F == kAny) {
    if (g.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = u.angle + i;
        if (j >= half) break;
        const float a = x[2 * i], b = x[2 * i + 1], c = cos[j], s = sin[j];
        x[2 * i] = a * c - b * s;
        x[2 * i + 1] = a * s + b * c;
      }
      return;
    }
    // (both values of a pair lie with lanes of one wave that come here, and a wave's LDS accesses keep their order)
#pragma unroll
    for (int i = 0; i < 16; ++i) row[u.at + i] = x[i];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = u.at + i;
      if (d >= 2 * half) break;
      const bool second = d >= half;
      const int j = second ? d - half : d;
      const float other = row[second ? j : d + half];
      x[i] = second ? other * sin[j] + x[i] * cos[j] : x[i] * cos[j] - other * sin[j];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    return;
  }
  cos += u.angle;
  sin += u.angle;
  constexpr bool INTERLEAVED = F == kNeighbours;
  const f32x4 c[2] = {__builtin_bit_cast(f32x4, load_16_bytes(cos)), __builtin_bit_cast(f32x4, load_16_bytes(cos + 4))};
  const f32x4 s[2] = {__builtin_bit_cast(f32x4, load_16_bytes(sin)), __builtin_bit_cast(f32x4, load_16_bytes(sin + 4))};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& u = x[INTERLEAVED ? 2 * i : i];
    float& v = x[INTERLEAVED ? 2 * i + 1 : 8 + i];
    const float a = u, b = v;
    u = a * c[i / 4][i % 4] - b * s[i / 4][i % 4];
    v = a * s[i / 4][i % 4] + b * c[i / 4][i % 4];
  }
}

constexpr int kMostTokens = 8, kMostThreads = 512;  // of a workgroup

// rows: tokens t0 .. t0 + count - 1, heads of q (if it is there), and of k and v with ALL
template <typename E, Form F, int D, bool ALL>
__device__ __forceinline__ void append_rows(const NormedArgs& a, int t0, int count, float (*weights)[D], float* values) {
  __shared__ Place places[kMostTokens];
  const gie_kv_geom& g = a.g;
  constexpr int L = kHeadLanes<D>;
  const int tid = int(threadIdx.x), threads = int(blockDim.x);
  for (int i = tid >> 6; i < count; i += threads >> 6) {
    const Place p = place_of(g, a.q_starts, a.seq_lens, a.page_table, t0 + i);
    if ((tid & 63) == 0) places[i] = p;
  }
  const Unit u = unit_of<F, D>(tid % L, g.rotary_dim);
  stage_weights<D>(a, weights);
  __syncthreads();
  const int q_heads = a.q ? g.q_heads : 0, heads = q_heads + (ALL ? 2 * g.kv_heads : 0), half = g.rotary_dim / 2;
#pragma unroll 2
  for (int i = tid / L; i < count * heads; i += threads / L) {
    const int j = i / heads, t = t0 + j;
    int head = i - j * heads;
    const Place p = places[j];
    const bool is_q = head < q_heads;
    if (!is_q) head -= q_heads;
    const bool is_v = !is_q && head >= g.kv_heads;
    if (is_v) head -= g.kv_heads;
    if (!p.present || (!is_q && p.page < 0)) continue;
    const uint16_t* src = (is_q ? a.q + t * g.q_stride : is_v ? a.v + t * g.v_stride : a.k + t * g.k_stride) + head * D;
    uint16_t* dst = is_q ? a.q_out + t * g.o_stride + head * D
                         : static_cast<uint16_t*>(is_v ? a.v_pages : a.k_pages) +
                               (((long long)p.page * g.kv_heads + head) * g.page_size + p.slot) * D;
    float x[16];
    load_unit<E>(src, u, x);
    if (is_q && a.q_norm) norm_unit<D>(x, weights[0], u, g.norm_eps);
    if (ALL && !is_q && !is_v && a.k_norm) norm_unit<D>(x, weights[1], u, g.norm_eps);
    if (u.pairs && !is_v && p.position >= 0)
      turn_unit<F>(x, u, g, a.cos + (long long)p.position * half, a.sin + (long long)p.position * half,
                   values + (F == kAny ? tid / L * L * 16 : 0));
    if (!u.there) continue;
    u32x4 y = {E::pack2(x[0], x[1]), E::pack2(x[2], x[3]), E::pack2(x[4], x[5]), E::pack2(x[6], x[7])};
    u32x4 z = {E::pack2(x[8], x[9]), E::pack2(x[10], x[11]), E::pack2(x[12], x[13]), E::pack2(x[14], x[15])};
    if (p.position < 0) y = z = u32x4{};
    store_16_bytes(dst + u.at, y);
    store_16_bytes(dst + u.next, z);
  }
}

// block `slot` of the batch's: a wave for each head of k and v, from `first_item` on
template <typename E, typename C, Form F, int D>
__device__ __forceinline__ void append_block(const NormedArgs& a, int slot, int first_item, float (*weights)[D],
                                             float* values) {
  const gie_kv_geom& g = a.g;
  constexpr int L = kHeadLanes<D>, T = 64 / L, kPasses = kKvBlock / T;  // T tokens at once
  const int tid = int(threadIdx.x), lane = tid & 63, half = g.rotary_dim / 2;
  const int item = first_item + __builtin_amdgcn_readfirstlane(tid >> 6);
  const Block b = block_of(g, a.q_starts, a.seq_lens, a.page_table, slot);
  if (b.first >= b.end || b.page < 0) return;
  if (a.k_norm) {
    stage_weights<D>(a, weights);
    __syncthreads();
  }
  const Unit u = unit_of<F, D>(lane % L, g.rotary_dim), straight = {lane % L * 16, lane % L * 16 + 8, 0, u.there, false};
  if (item < 2 * g.kv_heads) {
    const bool is_v = item >= g.kv_heads;
    const int head = is_v ? item - g.kv_heads : item;
    const long long stride = is_v ? g.v_stride : g.k_stride;
    const uint16_t* src = (is_v ? a.v : a.k) + b.row0 * stride + head * D;
    const long long at = ((long long)b.page * g.kv_heads + head) * g.page_size + b.slot;
    uint8_t* codes = static_cast<uint8_t*>(is_v ? a.v_pages : a.k_pages) + at * D;
    float* scale_at = (is_v ? a.v_scales : a.k_scales) + at / kKvBlock;
    const bool starts = b.first == b.start;
    const float before = starts ? 0.f : *scale_at;
    const Unit w = is_v ? straight : u;
    float x[kPasses][16];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int position = b.start + p * T + lane / L;
      if (position < b.first || position >= b.end) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[p][i] = 0.f;
        continue;
      }
      load_unit<E>(src + (position - b.first) * stride, w, x[p]);
    }
    if (!is_v && (a.k_norm || half > 0)) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int position = b.start + p * T + lane / L;
        if (position < b.first || position >= b.end) continue;
        if (a.k_norm) norm_unit<D>(x[p], weights[1], u, g.norm_eps);
        if (u.pairs)
          turn_unit<F>(x[p], u, g, a.cos + (long long)position * half, a.sin + (long long)position * half,
                       values + (F == kAny ? tid / L * L * 16 : 0));
      }
    }
    unsigned bits = 0;  // of the largest |x|: infinities and NaNs are larger than all numbers
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
      for (int i = 0; i < 16; ++i) bits = max(bits, __float_as_uint(x[p][i]) & 0x7fffffffu);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) bits = max(bits, unsigned(__shfl_xor(int(bits), d)));
    const float most = __uint_as_float(bits);
    if (bits >= 0x7f800000u || !(before == before)) {
      if (lane == 0) *scale_at = __builtin_nanf("");
      return;
    }
    const float scale = fmaxf(before, C::scale(most)), inv = 1.f / scale;
    const bool grows = !starts && scale > before;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int position = b.start + p * T + lane / L;
      uint8_t* dst = codes + (position - b.start) * D;
      if (!w.there || position >= b.end) continue;
      if (position < b.first) {
        if (!grows) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x2 c = __builtin_bit_cast(u32x2, *reinterpret_cast<const unsigned long long*>(dst + (i ? w.next : w.at)));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[p][8 * i + e] = C::decode1(c[e / 4] >> (e % 4 * 8) & 255u) * before;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[p][i] = C::divide(x[p][i], scale, inv);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x2 c = {C::encode4(x[p][8 * i], x[p][8 * i + 1], x[p][8 * i + 2], x[p][8 * i + 3]),
                         C::encode4(x[p][8 * i + 4], x[p][8 * i + 5], x[p][8 * i + 6], x[p][8 * i + 7])};
        *reinterpret_cast<unsigned long long*>(dst + (i ? w.next : w.at)) = __builtin_bit_cast(unsigned long long, c);
      }
    }
    if (lane == 0) *scale_at = scale;
  }
}

// C void: pages in the tokens' type. Otherwise the first `blocks` workgroups take blocks, `parts` of them one block's heads.
template <typename E, typename C, Form F, int D>
__global__ __launch_bounds__(kMostThreads) void append_kernel(NormedArgs a, int blocks, int parts, int tokens) {
  __shared__ __attribute__((aligned(16))) float weights[2][D];
  __shared__ __attribute__((aligned(16))) float values[F == kAny ? kMostThreads * 16 : 4];  // 16 of each lane
  int id = int(blockIdx.x);
  if constexpr (!std::is_void<C>::value) {
    if (id < blocks) {
      append_block<E, C, F, D>(a, id / parts, id % parts * (int(blockDim.x) >> 6), weights, values);
      return;
    }
    id -= blocks;
  }
  append_rows<E, F, D, std::is_void<C>::value>(a, id * tokens, min(tokens, a.g.total_tokens - id * tokens),
                                                         weights, values);
}

template <typename E, typename C>
int launch(const NormedArgs& a, hipStream_t s) {
  constexpr bool k8 = !std::is_void<C>::value;
  const gie_kv_geom& g = a.g;
  const int D = g.head_dim, lanes = D == 64 ? 4 : D == 256 ? 16 : 8;
  const long long heads = (a.q ? g.q_heads : 0) + (k8 ? 0 : 2 * g.kv_heads), work = heads * lanes;  // of a token's lanes
  // one token for each workgroup spreads a step of few tokens; of many, as many as give every lane two heads
  long long tokens = g.total_tokens < 1024 || work == 0 ? 1 : 1024 / work;
  tokens = tokens < 1 ? 1 : tokens > kMostTokens ? kMostTokens : tokens;
  // a wave looks places up one after the other: at most two
  while (tokens > 1 && tokens > 2 * ((work * tokens / 2 + 63) / 64)) tokens /= 2;
  const long long rows = heads == 0 ? 0 : (g.total_tokens + tokens - 1) / tokens;
  long long threads = (work * tokens + (tokens > 1 ? 127 : 63)) / (tokens > 1 ? 128 : 64) * 64;
  if (threads > kMostThreads) threads = kMostThreads;
  // blocks are a wave's work each: four waves to a workgroup spread them
  if (k8) threads = 256;
  const long long parts = (2ll * g.kv_heads + threads / 64 - 1) / (threads / 64), blocks = k8 ? block_slots(g) * parts : 0;
  if ((blocks + rows) * threads > 0xffffffffll) return GIE_HIP_EUNSUPPORTED;  // a launch's threads
  const auto kernel_of = [&](auto form) {
    constexpr Form F = decltype(form)::value;
    switch (D) {
      case 64: return append_kernel<E, C, F, 64>;
      case 96: return append_kernel<E, C, F, 96>;
      case 128: return append_kernel<E, C, F, 128>;
      default: return append_kernel<E, C, F, 256>;
    }
  };
  const auto kernel = g.rotary_dim % 16 != 0 ? kernel_of(std::integral_constant<Form, kAny>{})
                      : g.interleaved        ? kernel_of(std::integral_constant<Form, kNeighbours>{})
                                             : kernel_of(std::integral_constant<Form, kHalves>{});
  hipLaunchKernelGGL(kernel, dim3(unsigned(blocks + rows)),
                     dim3(unsigned(threads)), 0, s, a, int(blocks), int(parts), int(tokens));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

bool valid_rows(const gie_kv_geom* g, const void* q, const void* k, const void* v, const float* q_norm,
                const float* k_norm, const float* cos, const float* sin, const int* q_starts, const int* seq_lens,
                const int* page_table, const void* q_out, const void* k_pages, const void* v_pages) {
  if (!k || !v || !q_starts || !seq_lens || !page_table || !k_pages || !v_pages || k_pages == v_pages ||
      (q == nullptr) != (q_out == nullptr) || (q_norm && !q))
    return false;
  if (g->rotary_dim > 0 && (!cos || !sin || g->max_positions < (long long)g->max_pages * g->page_size)) return false;
  if (q == q_out && q && g->q_stride != g->o_stride) return false;
  if (!std::isfinite(g->norm_eps) || g->norm_eps < 0) return false;
  return aligned_to(q, 2) && aligned_to(k, 2) && aligned_to(v, 2) && aligned_to(q_out, 2) && aligned_to(k_pages, 16) &&
         aligned_to(v_pages, 16) && aligned_to(cos, 4) && aligned_to(sin, 4) && aligned_to(q_norm, 4) &&
         aligned_to(k_norm, 4);
}

bool supported(int dtype, const gie_kv_geom* g) {
  return (dtype == GIE_HIP_FP16 || dtype == GIE_HIP_BF16) &&
         (g->head_dim == 64 || g->head_dim == 96 || g->head_dim == 128 || g->head_dim == 256);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv_append_normed(int dtype, const gie_kv_geom* g, const void* q, const void* k, const void* v,
                                        const float* q_norm, const float* k_norm, const float* cos, const float* sin,
                                        const int* q_starts, const int* seq_lens, const int* page_table, void* q_out,
                                        void* k_pages, void* v_pages, void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (!q_norm && !k_norm) {
    const gie_paged_geom geom = narrowed(*g);
    return gie_hip_kv_append(dtype, &geom, q, k, v, cos, sin, q_starts, seq_lens, page_table, q_out, k_pages, v_pages, stream);
  }
  if (!supported(dtype, g)) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_rows(g, q, k, v, q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table, q_out, k_pages, v_pages))
    return GIE_HIP_EINVAL;
  const NormedArgs a{*g, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                     static_cast<const uint16_t*>(v), q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table,
                     static_cast<uint16_t*>(q_out), k_pages, v_pages, nullptr, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GIE_HIP_FP16 ? launch<Fp16, void>(a, s) : launch<Bf16, void>(a, s);
}

extern "C" int gie_hip_kv8_append(int dtype, int code, const gie_kv_geom* g, const void* q, const void* k,
                                  const void* v, const float* q_norm, const float* k_norm, const float* cos,
                                  const float* sin, const int* q_starts, const int* seq_lens, const int* page_table,
                                  void* q_out, void* k_pages, void* v_pages, float* k_scales, float* v_scales,
                                  void* stream) {
  if (!valid_paged(g) || !valid_code(code)) return GIE_HIP_EINVAL;
  if (!supported(dtype, g)) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_rows(g, q, k, v, q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table, q_out, k_pages, v_pages) ||
      !k_scales || !v_scales || k_scales == v_scales || !aligned_to(k_scales, 4) || !aligned_to(v_scales, 4))
    return GIE_HIP_EINVAL;
  const NormedArgs a{*g, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                     static_cast<const uint16_t*>(v), q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table,
                     static_cast<uint16_t*>(q_out), k_pages, v_pages, k_scales, v_scales};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool fp16 = dtype == GIE_HIP_FP16;
  if (code == GIE_HIP_KV_INT8) return fp16 ? launch<Fp16, Int8Code>(a, s) : launch<Bf16, Int8Code>(a, s);
  return fp16 ? launch<Fp16, E4m3Code>(a, s) : launch<Bf16, E4m3Code>(a, s);
}
