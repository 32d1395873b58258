// Attention of new tokens over a paged key/value cache held in 8 bits:
//   out[t][h] = sum_j p_j vs_j c^v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * ks_j * q[t][h] . c^k_j
// (or softcap * tanh(that / softcap)) with codes c and the scales ks, vs of position j's block of 16.
//
// One workgroup for each row (token, head), tiles of 64 keys: four lanes take a key's product, then every lane sums its
// value over the tile.
#include "attention_common.h"
#include "kv8_common.h"

namespace gie_hip {
namespace {

struct Kv8Args : AttnArgs {
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scales;
  const float* v_scales;
};

// a scale inside the range that the products assume; a NaN stays one
__device__ __forceinline__ float clamp_scale(float s) {
  return s == s ? fminf(fmaxf(s, 0x1p-73f), 0x1p120f) : s;
}

template <typename E, typename C>
__global__ __launch_bounds__(256) void rows_kernel(Kv8Args a, int D, float scale) {
  constexpr int TT = 64;
  __shared__ float q[256], weight[TT], top[4];
  const int tid = int(threadIdx.x);
  const int t = int(blockIdx.x) / a.q_heads, head = int(blockIdx.x) % a.q_heads, kvh = head / a.group;
  const Sequence seq = locate(a.q_starts, a.seq_lens, a.batch, a.total_tokens, t, [](int first, int) { return first; });
  if (t < seq.first || t >= seq.first + seq.count) return;
  int pos = seq.base + t - seq.first;
  if (pos >= a.capacity) pos = -1;
  const int oldest = a.window > 0 ? pos - a.window : -1;
  const KeyRange range = key_range<TT>(a, pos, pos);
  if (tid < D) q[tid] = E::to_f32(a.q[t * a.q_stride + head * D + tid]);
  const int page_size = a.page16 * 16;
  float m = -INFINITY, l = 0.f, o = 0.f;
  const auto at = [&](int key, bool& there) {  // of a key's codes, in heads of codes
    const int row = key / page_size, page = a.page_table[(long long)seq.index * a.max_pages + row];
    there = page >= 0 && page < a.num_pages;
    return ((long long)(there ? page : 0) * a.kv_heads + kvh) * page_size + (key - row * page_size);
  };
  for (int tile = 0; tile < range.tiles; ++tile) {
    const int key0 = tile < range.sink_tiles ? tile * TT : range.lo + (tile - range.sink_tiles) * TT;
    const int key = key0 + tid / 4;
    float s = -INFINITY;
    const bool seen = sees(a, key, pos, oldest);
    __syncthreads();
    float sum = 0.f;
    if (seen) {
      bool there;
      const long long from = at(key, there);
      if (there) {
        for (int d = tid % 4; d < D; d += 4) sum += q[d] * C::decode1(a.k_pages[from * D + d]);
        sum *= clamp_scale(a.k_scales[from / kKvBlock]);
      } else {
        for (int d = tid % 4; d < D; d += 4) sum += q[d] * 0.f;
      }
    }
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    if (seen) {
      s = sum * scale;
      if (a.cap > 0) s = a.cap * tanhf(s / a.cap);
    }
    float most = s;
#pragma unroll
    for (int d = 4; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if ((tid & 63) == 0) top[tid >> 6] = most;
    if (tid % 4 == 0) weight[tid / 4] = s;
    __syncthreads();
    const float next = fmaxf(fmaxf(m, fmaxf(top[0], top[1])), fmaxf(top[2], top[3]));
    const float ref = next == -INFINITY ? 0.f : next, keep = m == -INFINITY ? 1.f : expf(m - ref);
    m = next;
    l *= keep;
    o *= keep;
    for (int k = 0; k < TT; ++k) {
      if (!sees(a, key0 + k, pos, oldest)) continue;
      const float w = expf(weight[k] - ref);
      l += w;
      bool there;
      const long long from = at(key0 + k, there);
      if (there && tid < D)
        o += w * clamp_scale(a.v_scales[from / kKvBlock]) * C::decode1(a.v_pages[from * D + tid]);
    }
  }
  if (tid < D) a.out[t * a.o_stride + head * D + tid] = E::from_f32(l == 0.f ? 0.f : o / l);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_kv8_attention_workspace(const gie_paged_geom* g) { return 0; }

extern "C" int gie_hip_kv8_attention(int dtype, int code, const gie_paged_geom* g, const void* q, const void* k_pages,
                                     const void* v_pages, const float* k_scales, const float* v_scales,
                                     const int* q_starts, const int* seq_lens, const int* page_table, void* out,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_paged(g) || !valid_code(code)) return GIE_HIP_EINVAL;
  if (dtype != GIE_HIP_FP16 && dtype != GIE_HIP_BF16) return GIE_HIP_EUNSUPPORTED;
  if (g->head_dim != 64 && g->head_dim != 96 && g->head_dim != 128 && g->head_dim != 256) return GIE_HIP_EUNSUPPORTED;
  if (!std::isfinite(g->scale) || g->scale == 0 || !std::isfinite(g->softcap)) return GIE_HIP_EINVAL;
  if (g->total_tokens == 0) return GIE_HIP_OK;
  if (!valid_attention(g, q, k_pages, v_pages, q_starts, seq_lens, page_table, out)) return GIE_HIP_EINVAL;
  if (!k_scales || !v_scales || k_scales == v_scales || !aligned_to(k_scales, 4) || !aligned_to(v_scales, 4))
    return GIE_HIP_EINVAL;
  Kv8Args a{};
  a.k_pages = static_cast<const uint8_t*>(k_pages);
  a.v_pages = static_cast<const uint8_t*>(v_pages);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  Shape shape{};
  shape.splits = 1;
  shape.chunk = 1;
  fill_args(a, g, shape, q, q_starts, seq_lens, page_table, out, workspace);
  a.cap = g->softcap;
  const long long grid = (long long)g->total_tokens * g->q_heads;
  if (grid * 256 > 0xffffffffll) return GIE_HIP_EUNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto kernel = dtype == GIE_HIP_FP16
                          ? (code == GIE_HIP_KV_INT8 ? rows_kernel<Fp16, Int8Code> : rows_kernel<Fp16, E4m3Code>)
                          : (code == GIE_HIP_KV_INT8 ? rows_kernel<Bf16, Int8Code> : rows_kernel<Bf16, E4m3Code>);
  hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(256), 0, s, a, g->head_dim, g->scale);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
