// The keys and values of a batch's tokens out of an 8-bit paged cache, in the tokens' type: round(code * scale), with the
// scale of the head's block of 16 positions. Rows without a valid position or a page are zeros.
#include "kv8_common.h"

namespace gie_hip {
namespace {

struct ReadArgs {
  gie_paged_geom g;
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

template <typename E, typename C>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const gie_paged_geom& g = a.g;
  const int t = int(blockIdx.x), D = g.head_dim;
  const Place p = place_of(g, a.q_starts, a.seq_lens, a.page_table, t);
  if (!p.present) return;
  for (int i = int(threadIdx.x); i < 2 * g.kv_heads * D; i += 256) {
    const bool is_v = i >= g.kv_heads * D;
    const int c = is_v ? i - g.kv_heads * D : i, head = c / D, d = c - head * D;
    uint16_t* dst = is_v ? a.v : a.k;
    if (!dst) continue;
    float x = 0.f;
    if (p.page >= 0) {
      const long long at = ((long long)p.page * g.kv_heads + head) * g.page_size + p.slot;
      x = C::decode1((is_v ? a.v_pages : a.k_pages)[at * D + d]) * (is_v ? a.v_scales : a.k_scales)[at / kKvBlock];
    }
    dst[t * (is_v ? g.v_stride : g.k_stride) + c] = E::from_f32(x);
  }
}

template <typename E>
int launch(int code, const ReadArgs& a, hipStream_t s) {
  const auto kernel = code == GIE_HIP_KV_INT8 ? read_kernel<E, Int8Code> : read_kernel<E, E4m3Code>;
  hipLaunchKernelGGL(kernel, dim3(a.g.total_tokens), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv8_read(int dtype, int code, const gie_paged_geom* g, const void* k_pages, const void* v_pages,
                                const float* k_scales, const float* v_scales, const int* q_starts, const int* seq_lens,
                                const int* page_table, void* k, void* v, void* stream) {
  if (!valid_paged(g) || !valid_code(code)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0 || (!k && !v)) return GIE_HIP_OK;
  if (g->total_tokens > (1 << 24) - 1) return GIE_HIP_EUNSUPPORTED;  // a launch's threads
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
