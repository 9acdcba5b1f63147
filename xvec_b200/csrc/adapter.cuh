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

// A product and what is done with its sums.
//   kLinear: out = act(A B' + bias) + residual, save = A B' + bias
//   kGated:  out = act(A B0' + bias0) * (A B1' + bias1), save0 / save1 the two
//   kDx:     out = A0 B0 (+ A1 B1): gradients of the inputs
//   kDw:     out0 = A0' B, out1 = A1' B: gradients of the weights
enum Mode { kLinear = 0, kGated = 1, kDx = 2, kDw = 3 };

// One launch's parameters (adapter_gemm.cuh); the launch fills in the tiling.
struct GemmParams {
  int64_t rows, cols;    // of the output
  int tiles_m, tiles_n;  // tiles of the whole output
  int blocks;            // depth blocks of one product
  int segs;              // products added (kDx)
  int batches;           // outputs (kDw)
  int splits, blocks_per_split;  // of the segs * blocks depth blocks
  float* partial;        // splits > 1: [splits][batches or halves][rows][ldp] float sums
  int64_t ldp;
  uint32_t idesc;
  int vec;               // outputs, saves and residual allow 16-byte accesses
  const void* bias[2];
  const void* residual;
  void* out[2];
  void* save[2];
  int64_t ldr, ldo, lds;
  int act;
  int* status;
  uint64_t wait_ns;
};

// An operand in 16-bit elements: [planes][outer][inner], ld elements between
// rows (16 bytes or a multiple), plane elements between planes.
struct GemmOperand {
  const void* p = nullptr;
  int64_t inner = 0, outer = 0, ld = 0, plane = 0;
  int planes = 1;
};

// One product: rows, cols and the epilogue in p, sums over `depth` terms.
struct GemmCall {
  int mode = kLinear;
  bool bf16 = false;  // operands are bfloat16 (else binary16)
  int64_t depth = 0;
  GemmOperand a, b[2];
  GemmParams p{};
};
// By the storage type of the outputs; float32: operands are three bfloat16 planes.
xvec_gpu_status gemm_fp32(const GemmCall& c, cudaStream_t s);
xvec_gpu_status gemm_fp16(const GemmCall& c, cudaStream_t s);
xvec_gpu_status gemm_bf16(const GemmCall& c, cudaStream_t s);

}  // namespace adapter
}  // namespace xvec
