// Appends the keys and values of new tokens to a paged cache, rotating keys (and the tokens' queries) by their
// positions on the way:
//   pairs (u, v) = (x[j], x[j + R/2]) or (x[2j], x[2j+1]), j < R/2:  (u cos - v sin, u sin + v cos)
// with cos, sin = table[position][j] in FP32 and one rounding; the rest of a head is copied. Bytes-bound: every value
// is read once and written once, the tables' rows are shared by all heads of a token and come from the caches.
#include "paged_common.h"

namespace gie_hip {
namespace {

constexpr int kThreads = 256;

template <typename E>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(gie_paged_geom g, const uint16_t* q,
                                                             const uint16_t* __restrict__ k,
                                                             const uint16_t* __restrict__ v,
                                                             const float* __restrict__ cos_table,
                                                             const float* __restrict__ sin_table,
                                                             const int* __restrict__ q_starts,
                                                             const int* __restrict__ seq_lens,
                                                             const int* __restrict__ page_table,
                                                             uint16_t* q_out, uint16_t* __restrict__ k_pages,
                                                             uint16_t* __restrict__ v_pages) {
  const int t = int(blockIdx.x);
  const int b = find_sequence(g.batch, t, [&](int i) { return q_starts[i]; });
  const Rows rows = sequence_rows(q_starts, b, g.total_tokens);
  if (t < rows.first || t >= rows.first + rows.count) return;  // a row of no sequence
  const long long position = (long long)seq_lens[b] - rows.count + (t - rows.first);
  const bool placed = position >= 0 && position < (long long)g.max_pages * g.page_size;
  const int page = placed ? page_table[(long long)b * g.max_pages + position / g.page_size] : -1;
  const bool stored = page >= 0 && page < g.num_pages;
  const int slot = placed ? int(position % g.page_size) : 0;
  const int half = g.rotary_dim / 2, D = g.head_dim;
  const float* cos_row = cos_table + (placed ? position : 0) * half;
  const float* sin_row = sin_table + (placed ? position : 0) * half;
  const int heads = (q ? g.q_heads : 0) + 2 * g.kv_heads;
  const int units = D - half;  // of a head: pairs, then single values
  for (int i = threadIdx.x; i < heads * units; i += kThreads) {
    int head = i / units;
    const int u = i - head * units;
    const uint16_t* src;
    uint16_t* dst;
    bool turn = u < half, write;
    if (q && head < g.q_heads) {
      src = q + t * g.q_stride + head * D;
      dst = q_out + t * g.o_stride + head * D;
      write = true;
    } else {
      if (q) head -= g.q_heads;
      const bool is_v = head >= g.kv_heads;
      if (is_v) head -= g.kv_heads;
      src = (is_v ? v + t * g.v_stride : k + t * g.k_stride) + head * D;
      dst = (is_v ? v_pages : k_pages) + (((long long)page * g.kv_heads + head) * g.page_size + slot) * D;
      turn = turn && !is_v;
      write = stored;
    }
    if (!write) continue;
    const int at = u < half ? (g.interleaved ? 2 * u : u) : u + half;
    const int other = g.interleaved ? at + 1 : at + half;
    float a = E::to_f32(src[at]);
    if (u >= half) {
      dst[at] = placed ? src[at] : uint16_t(0);
    } else {
      float c = E::to_f32(src[other]);
      if (turn) {
        const float cs = cos_row[u], sn = sin_row[u];
        const float a2 = a * cs - c * sn;
        c = a * sn + c * cs;
        a = a2;
      }
      dst[at] = placed ? E::from_f32(a) : uint16_t(0);
      dst[other] = placed ? E::from_f32(c) : uint16_t(0);
    }
  }
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv_append(int dtype, const gie_paged_geom* g, const void* q, const void* k, const void* v,
                                 const float* cos, const float* sin, const int* q_starts, const int* seq_lens,
                                 const int* page_table, void* q_out, void* k_pages, void* v_pages, void* stream) {
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!k || !v || !q_starts || !seq_lens || !page_table || !k_pages || !v_pages || k_pages == v_pages ||
      (q == nullptr) != (q_out == nullptr))
    return GIE_HIP_EINVAL;
  if (g->rotary_dim > 0 && (!cos || !sin || g->max_positions < (long long)g->max_pages * g->page_size))
    return GIE_HIP_EINVAL;
  if (q == q_out && q && g->q_stride != g->o_stride) return GIE_HIP_EINVAL;
  if (!aligned_to(q, 2) || !aligned_to(k, 2) || !aligned_to(v, 2) || !aligned_to(q_out, 2) ||
      !aligned_to(k_pages, 16) || !aligned_to(v_pages, 16))
    return GIE_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto kernel = dtype == GIE_HIP_FP16 ? kv_append_kernel<Fp16> : kv_append_kernel<Bf16>;
  hipLaunchKernelGGL(kernel, dim3(g->total_tokens), dim3(kThreads), 0, s, *g, static_cast<const uint16_t*>(q),
                     static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), cos, sin, q_starts, seq_lens,
                     page_table, static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_pages),
                     static_cast<uint16_t*>(v_pages));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
