// Matrix product in 8-bit integers with one scale for each token and each output channel:
//   y[t,n] = round(act(float(sum_k q[t,k] * w[n,k]) * (x_scale[t] * w_scale[n]) + bias[n]))
// The sum is exact (int32), everything after it FP32 with one rounding to y's type. x is either given in 8 bits with
// its scales, or in the problem's precision; then each token's scale is found on the way:
//   a_t = max(max_k |x[t,k]|, 2^-100),  x_scale[t] = a_t / 127,  q[t,k] = rint(x[t,k] * (127 / a_t))
// A token that holds an infinity or a NaN gets scale NaN, so its whole row of y is NaN.
// Layouts: x is [tokens][in_features], w is [out_features][in_features], y is [tokens][out_features], rows ld elements
// apart. Calls only enqueue work on `stream`; the workspace is scratch of one call at a time.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "gpu_inference/conv2d.h"

namespace gie {

struct LinearI8Problem {
  int tokens = 1, in_features = 1, out_features = 1;
  Precision precision = Precision::kFp16;  // of x (unless quantized), bias and y: kFp32, kFp16 or kBf16
  bool has_bias = false;
  Activation activation = Activation::kNone;
  bool quantized = false;                // x is int8 with x_scale
  int64_t ld_x = 0, ld_w = 0, ld_y = 0;  // elements between rows; 0: packed
};

void validate_problem(const LinearI8Problem& prob);

class LinearI8 {
 public:
  // x_scale: null unless prob.quantized. workspace: 16-byte aligned, at least workspace_size(prob) bytes.
  static void forward(const void* x, const float* x_scale, const int8_t* w, const float* w_scale, const void* bias,
                      const LinearI8Problem& prob, void* y, void* workspace, size_t workspace_bytes,
                      hipStream_t stream);
  static size_t workspace_size(const LinearI8Problem& prob);
  // The quantization alone: q packed [tokens][in_features], scale [tokens].
  static void quantize_rows(const void* x, const LinearI8Problem& prob, int8_t* q, float* scale, hipStream_t stream);
};

}  // namespace gie
