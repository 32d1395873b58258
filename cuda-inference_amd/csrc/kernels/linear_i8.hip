// Matrix product in 8-bit integers with scales for each token and output channel:
//   y[t][n] = round(relu?(float(sum_k q[t][k] w[n][k]) * (x_scale[t] * w_scale[n]) + bias[n]))
#include "quantize_common.h"

namespace gie_hip {
namespace {

template <typename E>
__global__ __launch_bounds__(256) void linear_i8_kernel(const int8_t* __restrict__ x, const float* __restrict__ x_scale,
                                                        const int8_t* __restrict__ w, const float* __restrict__ w_scale,
                                                        const void* __restrict__ bias, void* __restrict__ y,
                                                        gie_linear_geom g) {
  const int n = int(blockIdx.x) * 64 + int(threadIdx.x & 63);
  const long long t = (long long)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (n >= g.out_features || t >= g.tokens) return;
  int acc = 0;
  for (int k = 0; k < g.in_features; ++k) acc += int(x[t * g.ld_x + k]) * int(w[n * g.ld_w + k]);
  float v = float(acc) * (x_scale[t] * w_scale[n]);  // the scales first: acc times a large one could pass FP32
  if (bias != nullptr) v += load_value<E>(bias, n);
  if (g.relu) v = v < 0.f ? 0.f : v;  // a NaN stays
  store_value<E>(y, t * g.ld_y + n, v);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

template <typename E>
void launch(const gie_linear_geom& g, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale,
            const void* bias, void* y, hipStream_t s) {
  hipLaunchKernelGGL(linear_i8_kernel<E>, dim3((g.out_features + 63) / 64, (g.tokens + 3) / 4), dim3(256), 0, s, x,
                     x_scale, w, w_scale, bias, y, g);
}

bool valid(int dtype, const gie_linear_geom* g) {
  return g && (dtype == GIE_HIP_FP32 || dtype == GIE_HIP_FP16 || dtype == GIE_HIP_BF16) && g->tokens >= 0 &&
         g->in_features > 0 && g->in_features <= 131071 && g->out_features > 0 && g->ld_x >= g->in_features &&
         g->ld_w >= g->in_features && g->ld_y >= g->out_features;
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" size_t gie_hip_linear_i8_workspace(int dtype, const gie_linear_geom* g, int quantized) {
  if (!valid(dtype, g) || quantized) return 0;
  return round16(size_t(g->tokens) * round16(g->in_features)) + round16(size_t(g->tokens) * 4);
}

extern "C" int gie_hip_linear_i8(int dtype, const gie_linear_geom* g, const void* x, const float* x_scale,
                                 const int8_t* w, const float* w_scale, const void* bias, void* y, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!valid(dtype, g)) return GIE_HIP_EINVAL;
  if (g->tokens == 0) return GIE_HIP_OK;
  if (!x || !w || !w_scale || !y || x == y) return GIE_HIP_EINVAL;
  const size_t esz = dtype == GIE_HIP_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(y) % esz != 0 || reinterpret_cast<uintptr_t>(bias) % esz != 0 ||
      reinterpret_cast<uintptr_t>(w_scale) % 4 != 0 || reinterpret_cast<uintptr_t>(x_scale) % 4 != 0)
    return GIE_HIP_EINVAL;
  const size_t need = gie_hip_linear_i8_workspace(dtype, g, x_scale != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return GIE_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  gie_linear_geom gg = *g;
  const int8_t* xq = static_cast<const int8_t*>(x);
  if (x_scale == nullptr) {
    int8_t* q = static_cast<int8_t*>(workspace);
    const size_t ld = round16(g->in_features);
    float* scale = reinterpret_cast<float*>(q + round16(g->tokens * ld));
    const int rc = gie_hip_quantize_rows(dtype, x, g->ld_x, g->tokens, g->in_features, q, ld, scale, stream);
    if (rc != GIE_HIP_OK) return rc;
    xq = q;
    x_scale = scale;
    gg.ld_x = int64_t(ld);
  }
  if (dtype == GIE_HIP_FP32)
    launch<F32>(gg, xq, x_scale, w, w_scale, bias, y, s);
  else if (dtype == GIE_HIP_FP16)
    launch<Fp16>(gg, xq, x_scale, w, w_scale, bias, y, s);
  else
    launch<Bf16>(gg, xq, x_scale, w, w_scale, bias, y, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
