// adapter.cuh — what the learned-adapter kernels share: element conversions,
// activations with their derivatives, and the products' descriptions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "capi_internal.h"

namespace xvec {
namespace adapter {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case XVEC_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);
    case XVEC_ACT_GELU: return 0.5f * z * (1.f + erff(z * kSqrtHalf));
    case XVEC_ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}
// act'(z).
__device__ __forceinline__ float slope(int act, float z) {
  switch (act) {
    case XVEC_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case XVEC_ACT_GELU:
      return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * expf(-0.5f * z * z) * kInvSqrt2Pi;
    case XVEC_ACT_SILU: {
      const float p = 1.f / (1.f + expf(-z));
      return p * (1.f + z * (1.f - p));
    }
    default: return 1.f;
  }
}

// Makes `device` current for one call and restores the caller's.
struct DeviceGuard {
  int before = -1;
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
  xvec_gpu_status set(int device);
};

// What a product does with its sums.
//   kLinear: out = act(A B' + bias) + residual, save = A B' + bias
//   kGated:  out = act(A B0' + bias0) * (A B1' + bias1), save0 / save1 the two
//   kDx:     out = A0 B0 (+ A1 B1): gradients of the inputs
//   kDw:     out0 = A0' B, out1 = A1' B: gradients of the weights
enum Mode { kLinear = 0, kGated = 1, kDx = 2, kDw = 3 };

// out [rows][cols] of one product, sums over `depth` terms.  a and b are the
// operands (two where the mode names two); their leading dimensions.
struct Product {
  int mode = kLinear;
  int storage = 0;
  int64_t rows = 0, cols = 0, depth = 0;
  int parts = 1;  // kDx: products added; kDw: outputs
  const void* a[2] = {};
  const void* b[2] = {};
  int64_t lda = 0, ldb = 0;
  const void* bias[2] = {};
  const void* residual = nullptr;
  void* out[2] = {};
  void* save[2] = {};
  int64_t ldr = 0, ldo = 0, lds = 0;
  int act = 0;
};

}  // namespace adapter
}  // namespace xvec
