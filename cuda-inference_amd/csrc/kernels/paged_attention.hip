// Attention of new tokens over a paged key/value cache:
//   out[t][h] = sum_j softmax_j(s_j) v_j,  s_j = scale * q[t][h] . k_j  (or softcap * tanh(that / softcap)),
// over the positions j <= p (and j > p - window) of the token's sequence. One wave for each row (token, head): the keys
// one after another with the running maximum and sum of the softmax.
#include "paged_common.h"

namespace gie_hip {
namespace {

template <typename E, int D>
__global__ __launch_bounds__(256) void attention_rows_kernel(gie_paged_geom g, const uint16_t* __restrict__ q,
                                                             const uint16_t* __restrict__ k_pages,
                                                             const uint16_t* __restrict__ v_pages,
                                                             const int* __restrict__ q_starts,
                                                             const int* __restrict__ seq_lens,
                                                             const int* __restrict__ page_table,
                                                             uint16_t* __restrict__ out) {
  constexpr int kPer = (D + 63) / 64;
  const int lane = int(threadIdx.x) & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long long)g.total_tokens * g.q_heads) return;
  const int t = int(row / g.q_heads), h = int(row % g.q_heads);
  const int b = find_sequence(g.batch, t, [&](int i) { return q_starts[i]; });
  const Rows rows = sequence_rows(q_starts, b, g.total_tokens);
  if (t < rows.first || t >= rows.first + rows.count) return;
  const long long capacity = (long long)g.max_pages * g.page_size;
  const long long position = (long long)seq_lens[b] - rows.count + (t - rows.first);
  const int kvh = h / (g.q_heads / g.kv_heads);
  float qv[kPer], acc[kPer];
  for (int i = 0; i < kPer; ++i) {
    const int d = i * 64 + lane;
    qv[i] = d < D ? E::to_f32(q[t * g.q_stride + h * D + d]) : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const long long last = position < capacity ? position : -1;  // a token without a valid position sees nothing
  const long long first = g.window > 0 && position - g.window + 1 > 0 ? position - g.window + 1 : 0;
  for (long long j = first; j <= last; ++j) {
    const int page = page_table[(long long)b * g.max_pages + j / g.page_size];
    const bool ok = page >= 0 && page < g.num_pages;
    const long long at = ((ok ? (long long)page : 0) * g.kv_heads + kvh) * g.page_size * D + (j % g.page_size) * D;
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) {
      const int d = i * 64 + lane;
      if (d < D) s += qv[i] * (ok ? E::to_f32(k_pages[at + d]) : 0.f);
    }
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    s *= g.scale;
    if (g.softcap > 0) s = g.softcap * tanhf(s / g.softcap);
    const float m2 = fmaxf(m, s);
    const float ref = m2 == -INFINITY ? 0.f : m2;  // scores of -infinity weigh nothing, a NaN stays one
    const float keep = __expf(m - ref);
    const float p = __expf(s - ref);
    m = m2;
    l = l * keep + p;
    for (int i = 0; i < kPer; ++i) {
      const int d = i * 64 + lane;
      acc[i] = acc[i] * keep + (d < D ? p * (ok ? E::to_f32(v_pages[at + d]) : 0.f) : 0.f);
    }
  }
  for (int i = 0; i < kPer; ++i) {
    const int d = i * 64 + lane;
    if (d < D) out[t * g.o_stride + h * D + d] = E::from_f32(l == 0.f ? 0.f : acc[i] / l);
  }
}

template <typename E>
int launch(const gie_paged_geom& g, const void* q, const void* k, const void* v, const int* q_starts,
           const int* seq_lens, const int* page_table, void* out, hipStream_t s) {
  const auto kernel = g.head_dim == 64    ? attention_rows_kernel<E, 64>
                      : g.head_dim == 96  ? attention_rows_kernel<E, 96>
                      : g.head_dim == 128 ? attention_rows_kernel<E, 128>
                                          : attention_rows_kernel<E, 256>;
  const long long rows = (long long)g.total_tokens * g.q_heads;
  hipLaunchKernelGGL(kernel, dim3(unsigned((rows + 3) / 4)), dim3(256), 0, s, g, static_cast<const uint16_t*>(q),
                     static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), q_starts, seq_lens, page_table,
                     static_cast<uint16_t*>(out));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_paged_attention_workspace(const gie_paged_geom* g) { return 0; }

extern "C" int gie_hip_paged_attention(int dtype, const gie_paged_geom* g, const void* q, const void* k_pages,
                                       const void* v_pages, const int* q_starts, const int* seq_lens,
                                       const int* page_table, void* out, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!q || !k_pages || !v_pages || !q_starts || !seq_lens || !page_table || !out || q == out) return GIE_HIP_EINVAL;
  if (!aligned_to(q, 2) || !aligned_to(out, 2) || !aligned_to(k_pages, 16) || !aligned_to(v_pages, 16))
    return GIE_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GIE_HIP_FP16 ? launch<Fp16>(*g, q, k_pages, v_pages, q_starts, seq_lens, page_table, out, s)
                               : launch<Bf16>(*g, q, k_pages, v_pages, q_starts, seq_lens, page_table, out, s);
}
