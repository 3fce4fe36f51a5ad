// Declarations shared by the C ABI of the quantised linear layer (api.cpp) and its kernels. All
// arguments are checked before these are called; everything a kernel needs travels by value.
#pragma once
#include <cstdint>

#include <cuda_runtime_api.h>

#include "immerdink/immerdink_linear.h"

namespace imd {

struct NormArgs {
  int64_t rows, dim;
  const void *x, *residual, *weight;
  void *residual_out, *q;
  float* scale;
  int64_t x_stride, residual_stride, residual_out_stride, q_stride;
  float eps, eps_root;             // eps and its square root (which keeps an eps below the 32-bit range)
  int32_t x_type, weight_type, q_type;
  unsigned int* error_word;
};
imd_status_t norm_quantize_launch(const NormArgs& a, cudaStream_t stream);

// A product out[t, n] of x [rows, k] and w [n, k]; `kind` is the weights' form.
enum class WeightKind : int32_t { kI8, kE4M3, kU4 };
struct LinearArgs {
  int64_t rows, n, k;
  const void *x, *w;
  int64_t x_stride, w_stride;      // elements; bytes for 4-bit weights
  const float *x_scale, *w_scale8; // 8-bit: one scale per row of x and of w
  const void* scale4;              // 4-bit: scales [n, groups], zeros [n, groups]
  const uint8_t* zeros;
  int64_t scale_stride, zeros_stride;
  void* out;
  int64_t out_stride;
  WeightKind kind;
  int32_t x_type, scale_type, out_type, group;
};
imd_status_t linear_small_launch(const LinearArgs& a, cudaStream_t stream);

}  // namespace imd
