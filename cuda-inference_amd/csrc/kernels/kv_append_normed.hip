// Appends the keys and values of new tokens to a paged cache as kv_append does, with a norm of each head of q and k ahead
// of the rotation, into pages of the tokens' own type or into 8-bit pages with a scale for each block of 16 positions:
//   x'_d = x_d / sqrt(mean_d x_d^2 + eps) * w_d;  pairs (u, v) -> (u cos - v sin, u sin + v cos);  FP32 up to one rounding.
#include <cmath>

#include "kv8_common.h"

namespace gie_hip {
namespace {

struct NormedArgs {
  gie_paged_geom g;
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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// One head by one wave: values lane, lane + 64, ... normed (w not null) and turned (position >= 0) in x; `row` is LDS of
// the wave's own for the pairs. The wave is its whole workgroup.
template <typename E>
__device__ __forceinline__ void head_values(const NormedArgs& a, const uint16_t* src, const float* w, bool turns,
                                            int position, float* row, float (&x)[4]) {
  const int D = a.g.head_dim, lane = int(threadIdx.x), rotary = a.g.rotary_dim, half = rotary / 2;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    x[i] = d < D ? E::to_f32(src[d]) : 0.f;
    sum += x[i] * x[i];
  }
  if (w != nullptr) {
    const float inv = 1.f / sqrtf(wave_sum(sum) / float(D) + a.g.norm_eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) x[i] = x[i] * inv * w[d];
    }
  }
  if (!turns || rotary == 0) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D) row[lane + 64 * i] = x[i];
  __syncthreads();
  const float* cos = a.cos + (long long)position * half;
  const float* sin = a.sin + (long long)position * half;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d >= rotary) continue;
    const bool second = a.g.interleaved ? d & 1 : d >= half;
    const int other = a.g.interleaved ? d ^ 1 : second ? d - half : d + half;
    const int j = a.g.interleaved ? d >> 1 : second ? d - half : d;
    x[i] = second ? row[other] * sin[j] + x[i] * cos[j] : x[i] * cos[j] - row[other] * sin[j];
  }
}

// one head of one token's q, and of its k and v where the pages hold the tokens' own type
template <typename E>
__global__ __launch_bounds__(64) void normed_rows_kernel(NormedArgs a, int heads) {
  __shared__ float row[256];
  const gie_paged_geom& g = a.g;
  const int t = int(blockIdx.x) / heads, lane = int(threadIdx.x), D = g.head_dim;
  int head = int(blockIdx.x) % heads;
  const Place p = place_of(g, a.q_starts, a.seq_lens, a.page_table, t);
  if (!p.present) return;
  const int q_heads = a.q ? g.q_heads : 0;
  const bool is_q = head < q_heads;
  if (!is_q && p.page < 0) return;
  if (!is_q) head -= q_heads;
  const bool is_v = !is_q && head >= g.kv_heads;
  if (is_v) head -= g.kv_heads;
  const uint16_t* src = is_q ? a.q + t * g.q_stride : is_v ? a.v + t * g.v_stride : a.k + t * g.k_stride;
  uint16_t* dst = is_q ? a.q_out + t * g.o_stride + head * D
                       : static_cast<uint16_t*>(is_v ? a.v_pages : a.k_pages) +
                             (((long long)p.page * g.kv_heads + head) * g.page_size + p.slot) * D;
  float x[4];
  head_values<E>(a, src + head * D, is_q ? a.q_norm : is_v ? nullptr : a.k_norm, !is_v && p.position >= 0, p.position, row, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) dst[d] = p.position < 0 ? uint16_t(0) : E::from_f32(x[i]);
  }
}

// one block of 16 positions of one key head's k or v
template <typename E, typename C>
__global__ __launch_bounds__(64) void block_values_kernel(NormedArgs a) {
  __shared__ float row[256];
  __shared__ float all[kKvBlock][256];
  const gie_paged_geom& g = a.g;
  const int items = 2 * g.kv_heads, D = g.head_dim, lane = int(threadIdx.x);
  const Block b = block_of(g, a.q_starts, a.seq_lens, a.page_table, int(blockIdx.x) / items);
  if (b.first >= b.end || b.page < 0) return;
  const int item = int(blockIdx.x) % items, head = item % g.kv_heads;
  const bool is_v = item >= g.kv_heads;
  const uint16_t* src = (is_v ? a.v + b.row0 * g.v_stride : a.k + b.row0 * g.k_stride) + head * D;
  const long long stride = is_v ? g.v_stride : g.k_stride;
  const long long at = ((long long)b.page * g.kv_heads + head) * g.page_size + b.slot;
  uint8_t* codes = static_cast<uint8_t*>(is_v ? a.v_pages : a.k_pages) + at * D;
  float* scale_at = (is_v ? a.v_scales : a.k_scales) + at / kKvBlock;
  float most = 0.f;
  bool finite = true;
  for (int p = b.first; p < b.end; ++p) {
    float x[4];
    head_values<E>(a, src + (p - b.first) * stride, is_v ? nullptr : a.k_norm, !is_v, p, row, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) continue;
      all[p - b.start][d] = x[i];
      most = fmaxf(most, fabsf(x[i]));
      finite = finite && fabsf(x[i]) <= 3.402823466e38f;
    }
  }
  most = wave_max(most);
  const bool starts = b.first == b.start;
  const float before = starts ? 0.f : *scale_at;
  if (__any(!finite) || !(before == before)) {
    if (lane == 0) *scale_at = __builtin_nanf("");
    return;
  }
  const float needed = C::scale(most), scale = fmaxf(before, needed), inv = 1.f / scale;
  if (!starts && scale > before)
    for (int p = b.start; p < b.first; ++p)
      for (int d = lane; d < D; d += 64) {
        uint8_t* c = codes + (p - b.start) * D + d;
        *c = uint8_t(C::encode1(C::decode1(*c) * (before * inv)));
      }
  for (int p = b.first; p < b.end; ++p)
    for (int d = lane; d < D; d += 64) codes[(p - b.start) * D + d] = uint8_t(C::encode1(all[p - b.start][d] * inv));
  if (lane == 0) *scale_at = scale;
}

bool valid_rows(const gie_paged_geom* g, const void* q, const void* k, const void* v, const float* q_norm,
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

bool supported(int dtype, const gie_paged_geom* g) {
  return (dtype == GIE_HIP_FP16 || dtype == GIE_HIP_BF16) &&
         (g->head_dim == 64 || g->head_dim == 96 || g->head_dim == 128 || g->head_dim == 256);
}

template <typename E, typename C>
int launch_blocks(const NormedArgs& a, hipStream_t s) {
  const long long grid = block_slots(a.g) * 2 * a.g.kv_heads;
  const long long rows = a.q ? (long long)a.g.total_tokens * a.g.q_heads : 0;
  if (grid * 64 > 0xffffffffll || rows * 64 > 0xffffffffll) return GIE_HIP_EUNSUPPORTED;  // a launch's threads
  hipLaunchKernelGGL((block_values_kernel<E, C>), dim3(unsigned(grid)), dim3(64), 0, s, a);
  if (rows > 0) hipLaunchKernelGGL(normed_rows_kernel<E>, dim3(unsigned(rows)), dim3(64), 0, s, a, a.g.q_heads);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_kv_append_normed(int dtype, const gie_paged_geom* g, const void* q, const void* k, const void* v,
                                        const float* q_norm, const float* k_norm, const float* cos, const float* sin,
                                        const int* q_starts, const int* seq_lens, const int* page_table, void* q_out,
                                        void* k_pages, void* v_pages, void* stream) {
  if (!q_norm && !k_norm)
    return gie_hip_kv_append(dtype, g, q, k, v, cos, sin, q_starts, seq_lens, page_table, q_out, k_pages, v_pages, stream);
  if (!valid_paged(g)) return GIE_HIP_EINVAL;
  if (!supported(dtype, g)) return GIE_HIP_EUNSUPPORTED;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_rows(g, q, k, v, q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table, q_out, k_pages, v_pages))
    return GIE_HIP_EINVAL;
  const NormedArgs a{*g, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                     static_cast<const uint16_t*>(v), q_norm, k_norm, cos, sin, q_starts, seq_lens, page_table,
                     static_cast<uint16_t*>(q_out), k_pages, v_pages, nullptr, nullptr};
  const long long heads = (q ? g->q_heads : 0) + 2 * g->kv_heads, grid = heads * g->total_tokens;
  if (grid * 64 > 0xffffffffll) return GIE_HIP_EUNSUPPORTED;  // a launch's threads
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GIE_HIP_FP16)
    hipLaunchKernelGGL(normed_rows_kernel<Fp16>, dim3(unsigned(grid)), dim3(64), 0, s, a, int(heads));
  else
    hipLaunchKernelGGL(normed_rows_kernel<Bf16>, dim3(unsigned(grid)), dim3(64), 0, s, a, int(heads));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}

extern "C" int gie_hip_kv8_append(int dtype, int code, const gie_paged_geom* g, const void* q, const void* k,
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
  if (code == GIE_HIP_KV_INT8) return fp16 ? launch_blocks<Fp16, Int8Code>(a, s) : launch_blocks<Bf16, Int8Code>(a, s);
  return fp16 ? launch_blocks<Fp16, E4m3Code>(a, s) : launch_blocks<Bf16, E4m3Code>(a, s);
}
