// The keys and values of a batch's tokens out of an 8-bit paged cache, in the tokens' type: round(code * scale), with the
// scale of the head's block of 16 positions. Rows without a valid position or a page are zeros.
//
// Bytes-bound: 16 codes in, 32 bytes out for each lane. A workgroup finds the places of one or more tokens and spreads all
// their heads over its lanes. 32768 tokens of 8 key heads of 128: 32 us alone, 47 among calls on other data (201 MB, 4.3
// TB/s; a large copy 4.7); one value for each lane and one token for each workgroup took 153.
#include "kv8_common.h"

namespace gie_hip {
namespace {

struct ReadArgs {
  gie_kv_geom g;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scales;
  const float* v_scales;
  const int* q_starts;
  const int* seq_lens;
  const int* page_table;
  uint16_t* k;
  uint16_t* v;
};

constexpr int kMostTokens = 8;  // of a workgroup

template <typename E, typename C, int D>
__global__ __launch_bounds__(512) void read_kernel(ReadArgs a, int tokens) {
  __shared__ Place places[kMostTokens];
  const gie_kv_geom& g = a.g;
  const int tid = int(threadIdx.x), threads = int(blockDim.x);
  const int t0 = int(blockIdx.x) * tokens, count = min(tokens, g.total_tokens - t0);
  for (int i = tid >> 6; i < count; i += threads >> 6) {
    const Place p = place_of(g, a.q_starts, a.seq_lens, a.page_table, t0 + i);
    if ((tid & 63) == 0) places[i] = p;
  }
  __syncthreads();
  constexpr int kUnits = D / 16;  // of 16 values
  const int units = 2 * g.kv_heads * kUnits;
#pragma unroll 2
  for (int i = tid; i < count * units; i += threads) {
    const int j = i / units, r = i - j * units, unit = r % kUnits;
    int head = r / kUnits;
    const bool is_v = head >= g.kv_heads;
    if (is_v) head -= g.kv_heads;
    const Place p = places[j];
    uint16_t* dst = is_v ? a.v : a.k;
    if (!p.present || !dst) continue;
    dst += (t0 + j) * (is_v ? g.v_stride : g.k_stride) + head * D + unit * 16;
    u32x4 y = {}, z = {};
    if (p.page >= 0) {
      const long long at = ((long long)p.page * g.kv_heads + head) * g.page_size + p.slot;
      const u32x4 c = *reinterpret_cast<const u32x4*>((is_v ? a.v_pages : a.k_pages) + at * D + unit * 16);
      const float scale = (is_v ? a.v_scales : a.k_scales)[at / kKvBlock];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const u32x2 v = C::decode4(c[w]);  // values 0 and 2, 1 and 3
        const auto value = [&](uint32_t x) { return Fp16::to_f32(uint16_t(x)) * C::kUnit * scale; };
        const uint32_t lo = E::pack2(value(v.x), value(v.y)), hi = E::pack2(value(v.x >> 16), value(v.y >> 16));
        if (w < 2)
          y[2 * w] = lo, y[2 * w + 1] = hi;
        else
          z[2 * w - 4] = lo, z[2 * w - 3] = hi;
      }
    }
    store_16_bytes(dst, y);
    store_16_bytes(dst + 8, z);
  }
}

template <typename E, typename C>
int launch(const ReadArgs& a, hipStream_t s) {
  const int D = a.g.head_dim, units = 2 * a.g.kv_heads * (D / 16);
  int tokens = a.g.total_tokens < 1024 ? 1 : 1024 / units;
  tokens = tokens < 1 ? 1 : tokens > kMostTokens ? kMostTokens : tokens;
  // a wave looks places up one after the other: at most two (1600 tokens of 2 key heads of 64: 6.4 us with eight)
  while (tokens > 1 && tokens > 2 * ((units * tokens / 2 + 63) / 64)) tokens /= 2;
  int threads = (units * tokens + 63) / 64 * 64;
  if (tokens > 1) threads = (units * tokens / 2 + 63) / 64 * 64;
  if (threads > 512) threads = 512;
  const auto kernel = D == 64 ? read_kernel<E, C, 64> : D == 96 ? read_kernel<E, C, 96> : D == 128 ? read_kernel<E, C, 128> : read_kernel<E, C, 256>;
  hipLaunchKernelGGL(kernel, dim3((a.g.total_tokens + tokens - 1) / tokens), dim3(threads), 0, s, a, tokens);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

template <typename E>
int launch(int code, const ReadArgs& a, hipStream_t s) {
  return code == GIE_HIP_KV_INT8 ? launch<E, Int8Code>(a, s) : launch<E, E4m3Code>(a, s);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv8_read(int dtype, int code, const gie_kv_geom* g, const void* k_pages, const void* v_pages,
                                const float* k_scales, const float* v_scales, const int* q_starts, const int* seq_lens,
                                const int* page_table, void* k, void* v, void* stream) {
  if (!valid_paged(g) || !valid_code(code)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0 || (!k && !v)) return GIE_HIP_OK;
  if (g->total_tokens > (1 << 23) - 1) return GIE_HIP_EUNSUPPORTED;  // 512 threads for each: a launch's limit
  if (!k_pages || !v_pages || !k_scales || !v_scales || !q_starts || !seq_lens || !page_table || k == v)
    return GIE_HIP_EINVAL;
  if (!aligned_to(k_pages, 16) || !aligned_to(v_pages, 16) || !aligned_to(k_scales, 4) || !aligned_to(v_scales, 4) ||
      !aligned_to(k, 2) || !aligned_to(v, 2))
    return GIE_HIP_EINVAL;
  const ReadArgs a{*g, static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), k_scales, v_scales,
                   q_starts, seq_lens, page_table, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GIE_HIP_FP16 ? launch<Fp16>(code, a, s) : launch<Bf16>(code, a, s);
}
