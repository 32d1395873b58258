// Device vocabulary of the 8-bit kernels (quantize_rows, linear_i8): loads of one value in storage type, a row's
// magnitude and scale, the rounding to 8 bits. Private to csrc/kernels.
#pragma once

#include "device_common.h"

namespace gie_hip {

struct F32 {  // 4-byte storage, no conversion
  static constexpr int kDtype = GIE_HIP_FP32;
};

template <typename E>
__device__ __forceinline__ float load_value(const void* p, long long i) {
  return E::to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <>
__device__ __forceinline__ float load_value<F32>(const void* p, long long i) {
  return static_cast<const float*>(p)[i];
}
template <typename E>
__device__ __forceinline__ void store_value(void* p, long long i, float v) {
  static_cast<uint16_t*>(p)[i] = E::from_f32(v);
}
template <>
__device__ __forceinline__ void store_value<F32>(void* p, long long i, float v) {
  static_cast<float*>(p)[i] = v;
}

// Magnitudes are compared as integers (the order of non-negative floats), where an infinity or a NaN is larger than
// every finite value and stays: a maximum in floating point would lose a NaN.
__device__ __forceinline__ float magnitude_max(float a, float v) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(v) & 0x7fffffffu));
}

__device__ __forceinline__ float wave_magnitude_max(float a) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) a = magnitude_max(a, __shfl_xor(a, d));
  return a;
}

// maximum over a workgroup of THREADS threads; every thread gets it
template <int THREADS>
__device__ __forceinline__ float block_magnitude_max(float a) {
  __shared__ float part[THREADS / 64];
  a = wave_magnitude_max(a);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  a = part[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) a = magnitude_max(a, part[i]);
  return a;
}

struct RowScale {
  float scale, inverse;
};
// `a`: the row's magnitude. The floor keeps 127 / a finite; a row of zeros gets q 0 from it. Both divisions are IEEE.
__device__ __forceinline__ RowScale row_scale(float a) {
  if (__float_as_uint(a) >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  a = fmaxf(a, 0x1p-100f);
  return {a / 127.f, 127.f / a};
}
// inverse 0 marks a row without a scale: its values (an infinity times 0 is a NaN) all become 0
__device__ __forceinline__ int8_t quantize_value(float v, float inverse) {
  return inverse == 0.f ? int8_t(0) : int8_t(int(rintf(v * inverse)));
}

// a 16-byte piece of a row: 8 values of 16 bits or 4 of 32
template <typename E>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = E::to_f32(uint16_t(v[e / 2] >> (16 * (e & 1))));
}
template <>
__device__ __forceinline__ void unpack<F32>(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[e]);
}
// ... and what it becomes, 8 or 4 bytes at `to` (any alignment)
template <typename E>
__device__ __forceinline__ void quantize_piece(u32x4 v, float inverse, void* to) {
  constexpr int kPer = E::kDtype == GIE_HIP_FP32 ? 4 : 8;
  float f[8];
  unpack<E>(v, f);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < kPer; ++e) w[e / 4] |= uint32_t(uint8_t(quantize_value(f[e], inverse))) << (8 * (e & 3));
  __builtin_memcpy(to, w, kPer);
}

}  // namespace gie_hip
