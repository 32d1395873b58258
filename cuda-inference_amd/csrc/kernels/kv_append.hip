// Appends the keys and values of new tokens to a paged cache, rotating keys (and the tokens' queries) by their
// positions on the way:
//   pairs (u, v) = (x[j], x[j + R/2]) or (x[2j], x[2j+1]), j < R/2:  (u cos - v sin, u sin + v cos)
// with cos, sin = table[position][j] in FP32 and one rounding; the rest of a head is copied.
//
// Bytes-bound: every value is read once and written once, the tables' rows are shared by all heads of a token and come
// from the caches. A thread takes 16 values of a head, 8 pairs where they rotate, in 16-byte pieces. A workgroup takes
// one or more whole tokens: a wave for each finds its sequence, position and page, then the threads go over all of the
// tokens' values. Heads whose rotating part is no multiple of 16 take a form that goes value by value.
//
// 8192 tokens of 32 + 2 x 8 heads of 128: 32 us, 6.4 TB/s (a large copy reaches 4.7: part of what is written stays in the
// caches); 64 tokens of one sequence each 3.6 us, which is a launch and the chain lengths -> page -> tables -> store. One
// value for each thread, and a search that loads one place after another, took 63 and 7.0 us.
#include "paged_common.h"

namespace gie_hip {
namespace {

constexpr int kMostTokens = 8;  // of a workgroup

struct AppendArgs {
  gie_paged_geom g;
  const uint16_t* q;  // null: only keys and values
  const uint16_t* k;
  const uint16_t* v;
  const float* cos;
  const float* sin;
  const int* q_starts;
  const int* seq_lens;
  const int* page_table;
  uint16_t* q_out;
  uint16_t* k_pages;
  uint16_t* v_pages;
  int tokens;  // of a workgroup
};

// where a token goes: position -1 without a valid one, page -1 if it is not stored, tokens of no sequence: absent
struct Place {
  int position, page, slot, present;
};

__device__ __forceinline__ Place place_of(const AppendArgs& a, int t) {
  const gie_paged_geom& g = a.g;
  const Sequence s = locate(a.q_starts, a.seq_lens, g.batch, g.total_tokens, t, [](int first, int) { return first; });
  Place p;
  p.present = t >= s.first && t < s.first + s.count;
  p.position = s.base + (t - s.first);
  if (!p.present || p.position < 0 || p.position >= g.max_pages * g.page_size) p.position = -1;
  p.page = -1;
  p.slot = 0;
  if (p.position >= 0) {
    const int row = p.position / g.page_size;
    const int page = a.page_table[(long long)s.index * g.max_pages + row];
    if (page >= 0 && page < g.num_pages) p.page = page;
    p.slot = p.position - row * g.page_size;
  }
  return p;
}

// a head's place in its source and its destination, for head `head` of a token's q, k and v heads one after another
struct Head {
  const uint16_t* src;
  uint16_t* dst;
  bool turns, stored;
};
__device__ __forceinline__ Head head_of(const AppendArgs& a, int t, int head, const Place& p) {
  const gie_paged_geom& g = a.g;
  const int D = g.head_dim, q_heads = a.q ? g.q_heads : 0;
  if (head < q_heads) return {a.q + t * g.q_stride + head * D, a.q_out + t * g.o_stride + head * D, true, true};
  head -= q_heads;
  const bool is_v = head >= g.kv_heads;
  if (is_v) head -= g.kv_heads;
  const long long at = (((long long)(p.page < 0 ? 0 : p.page) * g.kv_heads + head) * g.page_size + p.slot) * D;
  return {(is_v ? a.v + t * g.v_stride : a.k + t * g.k_stride) + head * D, (is_v ? a.v_pages : a.k_pages) + at, !is_v,
          p.page >= 0};
}

template <typename E, bool INTERLEAVED>
__device__ __forceinline__ void rotate8(u32x4& a, u32x4& b, const float* cos, const float* sin) {
  const f32x4 c0 = __builtin_bit_cast(f32x4, load_16_bytes(cos)), c1 = __builtin_bit_cast(f32x4, load_16_bytes(cos + 4));
  const f32x4 s0 = __builtin_bit_cast(f32x4, load_16_bytes(sin)), s1 = __builtin_bit_cast(f32x4, load_16_bytes(sin + 4));
  u32x4 x, y;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float ca = i < 4 ? c0[i] : c1[i - 4], cb = i < 4 ? c0[i + 1] : c1[i - 3];
    const float sa = i < 4 ? s0[i] : s1[i - 4], sb = i < 4 ? s0[i + 1] : s1[i - 3];
    if (INTERLEAVED) {  // pair i is word i of (a, b)
      const uint32_t wa = i < 4 ? a[i] : b[i - 4], wb = i < 4 ? a[i + 1] : b[i - 3];
      const float u0 = E::to_f32(uint16_t(wa)), v0 = E::to_f32(uint16_t(wa >> 16));
      const float u1 = E::to_f32(uint16_t(wb)), v1 = E::to_f32(uint16_t(wb >> 16));
      const uint32_t ra = E::pack2(u0 * ca - v0 * sa, u0 * sa + v0 * ca);
      const uint32_t rb = E::pack2(u1 * cb - v1 * sb, u1 * sb + v1 * cb);
      if (i < 4)
        x[i] = ra, x[i + 1] = rb;
      else
        y[i - 4] = ra, y[i - 3] = rb;
    } else {  // values i, i + 1 of a with those of b
      const float u0 = E::to_f32(uint16_t(a[i / 2])), v0 = E::to_f32(uint16_t(b[i / 2]));
      const float u1 = E::to_f32(uint16_t(a[i / 2] >> 16)), v1 = E::to_f32(uint16_t(b[i / 2] >> 16));
      x[i / 2] = E::pack2(u0 * ca - v0 * sa, u1 * cb - v1 * sb);
      y[i / 2] = E::pack2(u0 * sa + v0 * ca, u1 * sb + v1 * cb);
    }
  }
  a = x;
  b = y;
}

template <typename E, bool INTERLEAVED, int D>
__global__ __launch_bounds__(1024) void append_kernel(AppendArgs a) {
  __shared__ Place places[kMostTokens];
  const int tid = int(threadIdx.x), threads = int(blockDim.x);
  const int t0 = int(blockIdx.x) * a.tokens, count = min(a.tokens, a.g.total_tokens - t0);
  for (int i = tid >> 6; i < count; i += threads >> 6) {
    const Place p = place_of(a, t0 + i);
    if ((tid & 63) == 0) places[i] = p;
  }
  __syncthreads();
  constexpr int kUnits = D / 16;
  const int half = a.g.rotary_dim / 2, turning = a.g.rotary_dim / 16;
  const int units = ((a.q ? a.g.q_heads : 0) + 2 * a.g.kv_heads) * kUnits;
#pragma unroll 2
  for (int i = tid; i < count * units; i += threads) {
    const int j = i / units, u = i - j * units, head = u / kUnits, unit = u - head * kUnits;
    const Place p = places[j];
    if (!p.present) continue;
    const Head h = head_of(a, t0 + j, head, p);
    if (!h.stored) continue;
    const bool pairs = unit < turning;
    const int at = pairs && !INTERLEAVED ? unit * 8 : unit * 16;
    const int next = pairs && !INTERLEAVED ? at + half : at + 8;
    u32x4 x = load_16_bytes(h.src + at), y = load_16_bytes(h.src + next);
    if (pairs && h.turns && p.position >= 0)
      rotate8<E, INTERLEAVED>(x, y, a.cos + (long long)p.position * half + unit * 8,
                              a.sin + (long long)p.position * half + unit * 8);
    if (p.position < 0) x = u32x4{}, y = u32x4{};
    store_16_bytes(h.dst + at, x);
    store_16_bytes(h.dst + next, y);
  }
}

template <typename E>
__global__ __launch_bounds__(256) void append_values_kernel(AppendArgs a) {
  const int t = int(blockIdx.x);
  const Place p = place_of(a, t);
  if (!p.present) return;
  const int half = a.g.rotary_dim / 2, units = a.g.head_dim - half;  // of a head: pairs, then single values
  const int heads = (a.q ? a.g.q_heads : 0) + 2 * a.g.kv_heads;
  const float* cos = a.cos + (p.position < 0 ? 0 : (long long)p.position * half);
  const float* sin = a.sin + (p.position < 0 ? 0 : (long long)p.position * half);
  for (int i = threadIdx.x; i < heads * units; i += 256) {
    const int head = i / units, u = i - head * units;
    const Head h = head_of(a, t, head, p);
    if (!h.stored) continue;
    const int at = u < half && a.g.interleaved ? 2 * u : u < half ? u : u + half;
    if (u >= half) {
      h.dst[at] = p.position < 0 ? uint16_t(0) : h.src[at];
      continue;
    }
    const int other = a.g.interleaved ? at + 1 : at + half;
    uint16_t x = h.src[at], y = h.src[other];
    if (h.turns && p.position >= 0) {
      const float f = E::to_f32(x), g = E::to_f32(y);
      x = E::from_f32(f * cos[u] - g * sin[u]);
      y = E::from_f32(f * sin[u] + g * cos[u]);
    }
    h.dst[at] = p.position < 0 ? uint16_t(0) : x;
    h.dst[other] = p.position < 0 ? uint16_t(0) : y;
  }
}

template <typename E, bool INTERLEAVED>
auto kernel_for(int head_dim) {
  switch (head_dim) {
    case 64: return append_kernel<E, INTERLEAVED, 64>;
    case 96: return append_kernel<E, INTERLEAVED, 96>;
    case 128: return append_kernel<E, INTERLEAVED, 128>;
    default: return append_kernel<E, INTERLEAVED, 256>;
  }
}

template <typename E>
void launch(AppendArgs a, bool vec, hipStream_t s) {
  if (!vec) {
    hipLaunchKernelGGL(append_values_kernel<E>, dim3(a.g.total_tokens), dim3(256), 0, s, a);
    return;
  }
  const int units = ((a.q ? a.g.q_heads : 0) + 2 * a.g.kv_heads) * (a.g.head_dim / 16);
  // one token for each workgroup spreads a step of few tokens; of many, as many as give every thread two pieces of work
  int tokens = a.g.total_tokens < 1024 ? 1 : 1024 / units;
  tokens = tokens < 1 ? 1 : tokens > kMostTokens ? kMostTokens : tokens;
  a.tokens = tokens;
  int threads = (units * tokens + 63) / 64 * 64;
  if (tokens > 1) threads = (units * tokens / 2 + 63) / 64 * 64;
  if (threads > 512) threads = 512;
  const auto kernel = a.g.interleaved ? kernel_for<E, true>(a.g.head_dim) : kernel_for<E, false>(a.g.head_dim);
  hipLaunchKernelGGL(kernel, dim3((a.g.total_tokens + tokens - 1) / tokens), dim3(threads), 0, s, a);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv_append(int dtype, const gie_paged_geom* g, const void* q, const void* k, const void* v,
                                 const float* cos, const float* sin, const int* q_starts, const int* seq_lens,
                                 const int* page_table, void* q_out, void* k_pages, void* v_pages, void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (g->total_tokens > (1 << 23) - 1) return GIE_HIP_EUNSUPPORTED;  // 512 threads for each: a launch's limit
  if (!k || !v || !q_starts || !seq_lens || !page_table || !k_pages || !v_pages || k_pages == v_pages ||
      (q == nullptr) != (q_out == nullptr))
    return GIE_HIP_EINVAL;
  if (g->rotary_dim > 0 && (!cos || !sin || g->max_positions < (long long)g->max_pages * g->page_size))
    return GIE_HIP_EINVAL;
  if (q == q_out && q && g->q_stride != g->o_stride) return GIE_HIP_EINVAL;
  if (!aligned_to(q, 2) || !aligned_to(k, 2) || !aligned_to(v, 2) || !aligned_to(q_out, 2) ||
      !aligned_to(k_pages, 16) || !aligned_to(v_pages, 16) || !aligned_to(cos, 4) || !aligned_to(sin, 4))
    return GIE_HIP_EINVAL;
  const bool vec = g->rotary_dim % 16 == 0;
  AppendArgs a{*g, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
               cos, sin, q_starts, seq_lens, page_table, static_cast<uint16_t*>(q_out),
               static_cast<uint16_t*>(k_pages), static_cast<uint16_t*>(v_pages), 1};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GIE_HIP_FP16)
    launch<Fp16>(a, vec, s);
  else
    launch<Bf16>(a, vec, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
