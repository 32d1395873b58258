// Quantization of activations to 8 bits with one scale for each token (row):
//   a = max(max_k |x_k|, 2^-100), scale = a / 127, q_k = rint(x_k * (127 / a))
// in FP32 with nearest-even rounding; a row that holds an infinity or a NaN gets scale NaN and q 0, so that what is
// computed from it is NaN as well. HBM-bound: the row is read once from HBM and a second time from the cache.
#include "quantize_common.h"

namespace gie_hip {
namespace {

constexpr int kThreads = 256;

template <typename E>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const void* __restrict__ x, long long ld_x,
                                                                 int features, int8_t* __restrict__ q, long long ld_q,
                                                                 float* __restrict__ scale) {
  const long long row = blockIdx.x;
  const long long x0 = row * ld_x;
  float a = 0;
  for (int k = threadIdx.x; k < features; k += kThreads) a = magnitude_max(a, load_value<E>(x, x0 + k));
  a = block_magnitude_max<kThreads>(a);
  const RowScale s = row_scale(a);
  if (threadIdx.x == 0) scale[row] = s.scale;
  for (int k = threadIdx.x; k < features; k += kThreads)
    q[row * ld_q + k] = quantize_value(load_value<E>(x, x0 + k), s.inverse);
}

template <typename E>
void launch(const void* x, long long ld_x, int tokens, int features, int8_t* q, long long ld_q, float* scale,
            hipStream_t s) {
  hipLaunchKernelGGL(quantize_rows_kernel<E>, dim3(tokens), dim3(kThreads), 0, s, x, ld_x, features, q, ld_q, scale);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_quantize_rows(int dtype, const void* x, int64_t ld_x, int tokens, int features, int8_t* q,
                                     int64_t ld_q, float* scale, void* stream) {
  if (tokens < 0 || features <= 0 || ld_x < features || ld_q < features) return GIE_HIP_EINVAL;
  if (tokens == 0) return GIE_HIP_OK;
  if (!x || !q || !scale) return GIE_HIP_EINVAL;
  const size_t esz = dtype == GIE_HIP_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % esz != 0 || reinterpret_cast<uintptr_t>(scale) % 4 != 0) return GIE_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GIE_HIP_FP32)
    launch<F32>(x, ld_x, tokens, features, q, ld_q, scale, s);
  else if (dtype == GIE_HIP_FP16)
    launch<Fp16>(x, ld_x, tokens, features, q, ld_q, scale, s);
  else if (dtype == GIE_HIP_BF16)
    launch<Bf16>(x, ld_x, tokens, features, q, ld_q, scale, s);
  else
    return GIE_HIP_EUNSUPPORTED;
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GIE_HIP_OK : int(e);
}
