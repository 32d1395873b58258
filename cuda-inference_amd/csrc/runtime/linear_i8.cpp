// LinearI8: argument checks and the calls into the 8-bit kernels (gie_hip_linear_i8, gie_hip_quantize_rows).
#include "gpu_inference/linear_i8.h"

#include <string>

#include "gie_hip.h"
#include "gpu_inference/error.h"
#include "gpu_inference/roctx.h"

namespace gie {
namespace {

int dtype_of(Precision p) {
  return p == Precision::kFp16 ? GIE_HIP_FP16 : p == Precision::kBf16 ? GIE_HIP_BF16 : GIE_HIP_FP32;
}

gie_linear_geom geom_of(const LinearI8Problem& p) {
  gie_linear_geom g{};
  g.tokens = p.tokens;
  g.in_features = p.in_features;
  g.out_features = p.out_features;
  g.ld_x = p.ld_x ? p.ld_x : p.in_features;
  g.ld_w = p.ld_w ? p.ld_w : p.in_features;
  g.ld_y = p.ld_y ? p.ld_y : p.out_features;
  g.relu = p.activation == Activation::kReLU;
  return g;
}

void require(bool ok, const char* what) { GIE_REQUIRE(ok, StatusCode::kInvalidArgument, std::string("LinearI8: ") + what); }

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

void validate_problem(const LinearI8Problem& p) {
  require(p.tokens >= 0, "tokens must not be negative");
  require(p.in_features > 0 && p.out_features > 0, "features must be positive");
  require(p.ld_x == 0 || p.ld_x >= p.in_features, "ld_x is shorter than a row of x");
  require(p.ld_w == 0 || p.ld_w >= p.in_features, "ld_w is shorter than a row of w");
  require(p.ld_y == 0 || p.ld_y >= p.out_features, "ld_y is shorter than a row of y");
  GIE_REQUIRE(p.precision != Precision::kTf32, StatusCode::kUnsupported, "LinearI8: precision tf32 is not supported");
  GIE_REQUIRE(p.in_features <= 131071, StatusCode::kUnsupported,
              "LinearI8: more than 131071 input features could pass the range of the 32-bit sum");
}

size_t LinearI8::workspace_size(const LinearI8Problem& p) {
  validate_problem(p);
  const gie_linear_geom g = geom_of(p);
  return gie_hip_linear_i8_workspace(dtype_of(p.precision), &g, p.quantized ? 1 : 0);
}

void LinearI8::forward(const void* x, const float* x_scale, const int8_t* w, const float* w_scale, const void* bias,
                       const LinearI8Problem& p, void* y, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  validate_problem(p);
  if (p.tokens == 0) return;
  const size_t e = dtype_size(tensor_dtype(p.precision));
  require(x && w && w_scale && y, "x, w, w_scale and y must not be null");
  require(p.quantized == (x_scale != nullptr), "x_scale goes with quantized x, and only with it");
  require(p.has_bias == (bias != nullptr), "bias pointer and has_bias disagree");
  require(aligned(w_scale, 4) && aligned(x_scale, 4), "scales must be 4-byte aligned");
  require(aligned(y, e) && aligned(bias, e) && (p.quantized || aligned(x, e)),
          "x, bias and y must be aligned to their elements");
  require(x != y, "y must not be x");
  const gie_linear_geom g = geom_of(p);
  const int dtype = dtype_of(p.precision);
  const size_t need = gie_hip_linear_i8_workspace(dtype, &g, p.quantized ? 1 : 0);
  GIE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), StatusCode::kWorkspaceTooSmall,
              "LinearI8: workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(need) +
                  " needed");
  require(aligned(workspace, 16), "workspace must be 16-byte aligned");
  RoctxRange range("gie::LinearI8::forward");
  check_kernel_status(
      gie_hip_linear_i8(dtype, &g, x, x_scale, w, w_scale, bias, y, workspace, workspace_bytes, stream),
      "LinearI8::forward");
}

void LinearI8::quantize_rows(const void* x, const LinearI8Problem& p, int8_t* q, float* scale, hipStream_t stream) {
  validate_problem(p);
  if (p.tokens == 0) return;
  require(x && q && scale, "x, q and scale must not be null");
  require(aligned(x, dtype_size(tensor_dtype(p.precision))) && aligned(scale, 4),
          "x and scale must be aligned to their elements");
  check_kernel_status(gie_hip_quantize_rows(dtype_of(p.precision), x, p.ld_x ? p.ld_x : p.in_features, p.tokens,
                                            p.in_features, q, p.in_features, scale, stream),
                      "LinearI8::quantize_rows");
}

}  // namespace gie
