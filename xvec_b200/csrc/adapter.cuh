// adapter.cuh — what the learned-adapter kernels share: element conversions,
// activations with their derivatives, and the products' descriptions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

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

// Two values side by side, each rounded to T.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (sizeof(T) != 2) return 0;
  uint32_t u;
  if constexpr (std::is_same<T, bf16>::value) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    memcpy(&u, &t, 4);
  } else {
    const __half2 t = __floats2half2_rn(a, b);
    memcpy(&u, &t, 4);
  }
  return u;
}

constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// exp(-x) for x >= 0: the 16-bit types' form is off by x 2^-23 relative to itself.
template <typename T>
__device__ __forceinline__ float exp_minus(float x) {
  return sizeof(T) == 4 ? expf(-x) : __expf(-x);
}

// Phi(z), the standard normal distribution, and *gauss = exp(-z^2 / 2).  For a = |z|:
//   Phi(-a) = exp(-a^2 / 2) R(a),  R(a) = erfc(a / sqrt 2) exp(a^2 / 2) / 2 = t P(t),
//   t = 1 / (1 + 39/128 a),
// P of degree 7, fitted to R on a = 0..14.5 for the least largest relative error (1.0e-7).  So
// the far negative tail, where gelu is small, keeps its relative accuracy: evaluated in
// float32 Phi(-a) is off by 4.3e-7 of itself at most (a <= 12; the 16-bit exponential
// adds a^2 2^-24), and Phi(a) by 2.2e-7.  float32 makes up for the rounding of a^2.  With
// erff the epilogue was the longest part of a tile (float32 10000 x 960 -> 960 149 us).
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
  // (At 16 both are 0; an infinite square would have no rounding to make up for.)
  const float a = fminf(fabsf(z), 16.f), s = a * a;
  float e = exp_minus<T>(0.5f * s);
  if (sizeof(T) == 4) e = fmaf(-0.5f * fmaf(a, a, -s), e, e);
  const float t = __fdividef(1.f, fmaf(0.3046875f, a, 1.f));
  float q = fmaf(0.036564309f, t, -0.15296334f);
  q = fmaf(q, t, 0.18648443f);
  q = fmaf(q, t, -0.038461823f);
  q = fmaf(q, t, 0.12123448f);
  q = fmaf(q, t, 0.10327935f);
  q = fmaf(q, t, 0.12234776f);
  q = fmaf(q, t, 0.12151483f);
  const float tail = q * t * e;
  *gauss = e;
  return z < 0.f ? tail : 1.f - tail;
}
// 1 / (1 + exp(-z)), and its difference to 1 in *rest.  The fast quotient is 0 for divisors
// above 2^126 (z below -87.3), which bfloat16's and float32's small results would
// notice: bfloat16 divides both sides by 2^8; float32, which has no bits to lose in the
// exponential's argument, takes exp(-|z|), and so has *rest without cancellation.
template <typename T>
__device__ __forceinline__ float sigmoid(float z, float* rest) {
  constexpr float kLog256 = 5.5451774f, kBy256 = 0.00390625f;
  if constexpr (sizeof(T) == 2) {
    const float s = std::is_same<T, bf16>::value
                        ? __fdividef(kBy256, kBy256 + __expf(-z - kLog256))
                        : __fdividef(1.f, 1.f + __expf(-z));
    *rest = 1.f - s;
    return s;
  }
  const float e = exp_minus<T>(fabsf(z)), r = __fdividef(1.f, 1.f + e), er = e * r;
  *rest = z < 0.f ? r : er;
  return z < 0.f ? er : r;
}

template <typename T>
__device__ __forceinline__ float relu(float z) {
  return z > 0.f ? z : (z == z ? 0.f : z);
}
template <typename T>
__device__ __forceinline__ float gelu(float z) {
  float e;
  return z * normal_cdf<T>(z, &e);
}
template <typename T>
__device__ __forceinline__ float silu(float z) {
  float rest;
  return z * sigmoid<T>(z, &rest);
}

// act(z) for results of type T.
template <typename T>
__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case XVEC_ACT_RELU: return relu<T>(z);
    case XVEC_ACT_GELU: return gelu<T>(z);
    case XVEC_ACT_SILU: return silu<T>(z);
    default: return z;
  }
}
template <typename T, int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
  if (act == XVEC_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = relu<T>(v[j]);
  } else if (act == XVEC_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gelu<T>(v[j]);
  } else if (act == XVEC_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = silu<T>(v[j]);
  }
}
// act(z), and act'(z) in *slope.
template <typename T>
__device__ __forceinline__ float activate_slope(int act, float z, float* slope) {
  switch (act) {
    case XVEC_ACT_RELU:
      *slope = z > 0.f ? 1.f : 0.f;
      return relu<T>(z);
    case XVEC_ACT_GELU: {
      float e;
      const float cdf = normal_cdf<T>(z, &e);
      *slope = fmaf(z * e, kInvSqrt2Pi, cdf);
      return z * cdf;
    }
    case XVEC_ACT_SILU: {
      float rest;
      const float s = sigmoid<T>(z, &rest);
      *slope = s * fmaf(z, rest, 1.f);
      return z * s;
    }
    default:
      *slope = 1.f;
      return z;
  }
}

// Sixteen bytes that start `off` bytes into granule a and end in the next, b:
// selects by the offset's words, then a funnel shift by its half word.
template <typename T>
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, uint32_t off) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
  if (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The 16-byte granule at p, if it starts before `end`.  A plain load, as everywhere in
// these kernels: they are resident before the launch that writes their inputs has
// completed (pdl_wait), and a non-coherent load needs memory that does not change
// while its kernel runs.
__device__ __forceinline__ uint4 granule(uintptr_t p, uintptr_t end) {
  return p < end ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

// Eight elements of a row, of which `count` exist (what the others hold is of no
// account), in two steps: load requests the 16-byte granules that hold them, each
// only if it holds one of the elements; settle, once they are needed, shifts
// them together where they do not start on 16 bytes (VEC: they do).
template <typename T, bool VEC>
struct Eight {
  static constexpr int N = sizeof(T) / 2;  // 16-byte parts
  uint4 v[VEC ? N : N + 1];
  uint32_t off;
  __device__ __forceinline__ void load(const T* p, int count) {
    off = VEC ? 0 : (uint32_t)(uintptr_t)p & 15;
    const uintptr_t base = (uintptr_t)p - off;
    const uintptr_t end = (uintptr_t)(p + (count < 8 ? count : 8));
#pragma unroll
    for (int i = 0; i < (VEC ? N : N + 1); ++i) v[i] = granule(base + 16 * i, end);
  }
  __device__ __forceinline__ void settle() {
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = shifted<T>(v[i], v[i + 1], off);
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    return to_f(reinterpret_cast<const T*>(v)[j]);
  }
};

// Launches of one call overlap at their edges: a kernel is started while the one
// before it still runs, touches memory only once that has completed (pdl_wait),
// and then lets the next be started as soon as all its own blocks are there
// (pdl_launch).  Worth 2 to 3 us for each launch of a call that has several.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_begin() {
  pdl_wait();
  pdl_launch();
}
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kern)(Params...), dim3 grid, int block, size_t smem, cudaStream_t s,
                       int cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
  if (e == cudaSuccess) XVEC_LAUNCHED();
  return e;
}

// Makes `device` current for one call and restores the caller's.  Meanwhile a
// stream capture of another thread does not forbid the one-time settings and the
// loading of kernels (none of them belongs into a graph).
struct DeviceGuard {
  cudaMemPool_t pool = nullptr;  // the device's scratch
  int before = -1;
  bool relaxed = false;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  ~DeviceGuard();
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
  float* runs;           // float32, long sums: those of finished runs, by thread
  const float* scale;    // what sums are multiplied by (binary16 kDx, kDw; may be NULL)
  uint32_t idesc;
  int vec;               // bytes of an access that outputs and saves allow
  int bias_vec;          // the biases allow 16
  const void* bias[2];
  const void* residual;
  void* out[2];
  void* save[2];
  int64_t ldr, ldo, lds;
  int act;
  // Column sums for the warps that have no part in the product (column_sums).
  const float* sums;
  int sum_chunks, sum_cols;
  void* sum_out[2];
  // This launch may run beside the one before it, which it shares nothing with but
  // inputs that were complete when that one began (its pdl_launch came after its
  // pdl_wait): it waits for it at its own end instead, so that whatever comes
  // later still finds both complete.
  int beside;
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
  int device = 0, sms = 0;    // (plan_gemm)
  int shape = 0;              // of the tiles (plan_gemm)
  size_t partial_bytes = 0;   // scratch for split sums, at p.partial
  size_t run_bytes = 0;       // scratch for float32's long sums, at p.runs
};
// Depth blocks of 64 that one accumulation takes (adapter_gemm.cuh): 16-bit storage 2048
// terms, float32 4096 (whose large products leave the accumulator far more often).
constexpr int run_blocks(bool float32) { return float32 ? 64 : 32; }
constexpr int kShapes = 4;
struct TileShape {
  int rows, cols;  // cols: of the accumulator (half as many outputs when gated)
  bool pair;
};
constexpr TileShape kTileShapes[kShapes] = {
    {256, 256, true}, {256, 192, true}, {256, 128, true}, {128, 128, false}};
// Picks the tiles and splits: fills in c's tiling and its scratch.
xvec_gpu_status plan_gemm(int storage, GemmCall* c);
// The number of SMs of a device.
xvec_gpu_status count_sms(int device, int* sms);
// By the storage type of the outputs; float32: operands are three bfloat16 planes.
xvec_gpu_status gemm_fp32(const GemmCall& c, cudaStream_t s);
xvec_gpu_status gemm_fp16(const GemmCall& c, cudaStream_t s);
xvec_gpu_status gemm_bf16(const GemmCall& c, cudaStream_t s);

// out[o][c] = the sum over the chunks of sums[o][chunk][c], o = 0, 1, in a fixed
// order: four interleaved runs, then those.  Warp `worker` of `workers` takes
// every workers-th group of 8 columns.
template <typename T>
__device__ __forceinline__ void column_sums(const float* sums, int chunks, int m, void* out0,
                                            void* out1, int worker, int workers, int lane) {
  const int groups = (m + 7) / 8;
  for (int g = worker; g < 2 * groups; g += workers) {
    T* out = static_cast<T*>(g < groups ? out0 : out1);
    if (!out) continue;
    const int c = (g < groups ? g : g - groups) * 8 + (lane & 7);
    const float* p = sums + (g < groups ? 0 : (int64_t)chunks * m) + c;
    float s = 0.f;
    if (c < m) {
#pragma unroll 8
      for (int i = lane >> 3; i < chunks; i += 4) s += p[(int64_t)i * m];
    }
    s += __shfl_xor_sync(0xffffffffu, s, 8);
    s += __shfl_xor_sync(0xffffffffu, s, 16);
    if (lane < 8 && c < m) out[c] = from_f<T>(s);
  }
}

// The widest access in bytes, up to 16, that fits every row.
inline int access_width(const void* p, int64_t ld, size_t size) {
  const uint64_t bits = 16 | (uintptr_t)p | (uint64_t)ld * size;
  return (int)(bits & (~bits + 1));
}
// Rows read in place with 16-byte accesses.
inline bool aligned16(const void* p, int64_t ld, size_t size) {
  return (uintptr_t)p % 16 == 0 && ld * (int64_t)size % 16 == 0;
}

// The forward calls for a few rows (adapter_few.cu): kLinear, or with two weights kGated.
// Whether they go through few_rows.  Estimates in us, M = millions of weights,
// for each eight rows: few rows 0.65 M (16-bit, up to four rows), 3 M (more), 0.95 M
// and 1.2 M (float32); the matrix kernel 9.6 + 0.2 M, and for float32, whose
// weights it has to split first, 15 + 3.3 M.  Measured, 1024 x 1024 fp16: 4 rows 2.9
// against 9.5, 16 rows 4.4 against 9.5; 4096 x 4096: 4 rows 12.5 against 12.8, 8 rows
// 22.8 against 12.8; fp32 8 rows 20.5 against 70.
inline bool use_few_rows(int storage, int64_t n, int64_t in_dim, int64_t out_dim, int weights) {
  if (n > 64) return false;
  const double m = 1e-6 * (double)in_dim * (double)out_dim * weights;
  const double groups = (double)((n + 7) / 8);
  return storage == XVEC_STORAGE_FP32 ? groups * (n <= 4 ? 0.95 : 1.2) * m < 15 + 3.3 * m
                                      : groups * (n <= 4 ? 0.65 : 3.0) * m < 9.6 + 0.2 * m;
}
struct FewRows {
  int n, in_dim, out_dim, act;
  const void *x, *w[2], *bias[2], *residual;
  void *out, *save[2];
  int64_t ldx, ldw, ldr, ldo, lds;
};
xvec_gpu_status few_rows(int storage, const FewRows& f, cudaStream_t s);

}  // namespace adapter
}  // namespace xvec
