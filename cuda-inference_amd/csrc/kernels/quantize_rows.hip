// Quantization of activations to 8 bits with one scale for each token (row):
//   a = max(max_k |x_k|, 2^-100), scale = a / 127, q_k = rint(x_k * (127 / a))
// in FP32 with nearest-even rounding; a row that holds an infinity or a NaN gets scale NaN and q 0, so that what is
// computed from it is NaN as well. HBM-bound: a row is read once, in 16-byte pieces that its threads keep in
// registers between the maximum and the rounding; what passes the registers is read a second time from the cache.
// A wave takes a row of up to 2048 bytes (four rows for each workgroup), a workgroup a longer one. 4096 rows of 4096 FP16
// values: 10.6 to 11.2 us, 4.5 to 4.7 TB/s (read and written), the rate of a large copy; 64 rows of 8192 2.9 us, a launch.
#include "quantize_common.h"

namespace gie_hip {
namespace {

constexpr int kThreads = 256, kKeep = 4;

// T threads for each row; rows of x and q of any alignment
template <typename E, int T>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const void* __restrict__ x, long long ld_x, int tokens,
                                                                 int features, int8_t* __restrict__ q, long long ld_q,
                                                                 float* __restrict__ scale) {
  constexpr int kE = E::kDtype == GIE_HIP_FP32 ? 4 : 2, kPer = 16 / kE;
  const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / T) + threadIdx.x / T;
  const bool there = row < tokens;  // a wave without a row still meets the others' barriers
  const int me = int(threadIdx.x) % T;
  const long long x0 = there ? row * ld_x : 0;
  const int pieces = there ? features / kPer : 0;  // whole ones; the rest value by value
  const int rest = there ? pieces * kPer : features;
  const char* xv = static_cast<const char*>(x) + x0 * kE;
  float a = 0;
  u32x4 keep[kKeep];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) keep[i] = i * T + me < pieces ? load_16_bytes(xv + (i * T + me) * 16ll) : u32x4{};
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    float f[8];
    unpack<E>(keep[i], f);
#pragma unroll
    for (int e = 0; e < kPer; ++e) a = magnitude_max(a, f[e]);
  }
  for (int p = kKeep * T + me; p < pieces; p += T) {
    float f[8];
    unpack<E>(load_16_bytes(xv + p * 16ll), f);
#pragma unroll
    for (int e = 0; e < kPer; ++e) a = magnitude_max(a, f[e]);
  }
  for (int k = rest + me; k < features; k += T) a = magnitude_max(a, load_value<E>(x, x0 + k));
  a = T == 64 ? wave_magnitude_max(a) : block_magnitude_max<kThreads>(a);
  const RowScale s = row_scale(a);
  if (me == 0 && there) scale[row] = s.scale;
  int8_t* out = q + (there ? row * ld_q : 0);
  const auto put = [&](int p, u32x4 v) { quantize_piece<E>(v, s.inverse, out + p * kPer); };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (i * T + me < pieces) put(i * T + me, keep[i]);
  for (int p = kKeep * T + me; p < pieces; p += T) put(p, load_16_bytes(xv + p * 16ll));
  for (int k = rest + me; k < features; k += T) out[k] = quantize_value(load_value<E>(x, x0 + k), s.inverse);
}

template <typename E>
void launch(const void* x, long long ld_x, int tokens, int features, int8_t* q, long long ld_q, float* scale, hipStream_t s) {
  constexpr int kE = E::kDtype == GIE_HIP_FP32 ? 4 : 2;
  const bool small = features <= 64 * 16 * 2 / kE;
  const int blocks = small ? tokens / 4 + (tokens % 4 != 0) : tokens, across = blocks < (1 << 20) ? blocks : 1 << 20;
  const auto kernel = small ? quantize_rows_kernel<E, 64> : quantize_rows_kernel<E, kThreads>;
  hipLaunchKernelGGL(kernel, dim3(across, blocks / across + (blocks % across != 0)), dim3(kThreads), 0, s, x, ld_x, tokens, features,
                     q, ld_q, scale);
}

}  // namespace
}  // namespace gie_hip

using namespace gie_hip;

extern "C" int gie_hip_quantize_rows(int dtype, const void* x, int64_t ld_x, int tokens, int features, int8_t* q,
                                     int64_t ld_q, float* scale, void* stream) {
  if (tokens < 0 || features <= 0 || ld_x < features || ld_q < features) return GIE_HIP_EINVAL;
  if (features > (1 << 30)) return GIE_HIP_EUNSUPPORTED;  // a step past the row's end still has to fit 32 bits
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
