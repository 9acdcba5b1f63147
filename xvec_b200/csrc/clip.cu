// clip.cu — the global norm of many gradient tensors and their clipping to it.
//
//   norm = sqrt(sum over all tensors of x^2),  out = x min(1, max_norm / norm)
//
// Bound by memory: every element is read once for the norm and once for the
// scaling, and written once.  The tensors are cut into chunks of kChunk
// elements; a block owns whole chunks, so the order of the sums depends on the
// sizes alone and results repeat.
#include <algorithm>
#include <cmath>
#include <new>

#include "adapter.cuh"

namespace xvec {
namespace adapter {
namespace {

constexpr int kChunk = 16384;  // elements
constexpr int kThreads = 256;
constexpr int kMaxEntries = 500;  // per launch: the table travels as a kernel parameter

struct Entry {
  const void* in;
  void* out;
  int64_t count;
  int32_t storage;
  uint32_t first_chunk;  // of this launch
};
struct Table {
  int entries;
  uint32_t chunks;
  Entry e[kMaxEntries];
};

__device__ __forceinline__ float load_as_float(const Entry& e, int64_t i) {
  switch (e.storage) {
    case XVEC_STORAGE_FP32: return static_cast<const float*>(e.in)[i];
    case XVEC_STORAGE_FP16: return to_f(static_cast<const __half*>(e.in)[i]);
    default: return to_f(static_cast<const bf16*>(e.in)[i]);
  }
}
__device__ __forceinline__ void store_from_float(const Entry& e, int64_t i, float v) {
  switch (e.storage) {
    case XVEC_STORAGE_FP32: static_cast<float*>(e.out)[i] = v; break;
    case XVEC_STORAGE_FP16: static_cast<__half*>(e.out)[i] = from_f<__half>(v); break;
    default: static_cast<bf16*>(e.out)[i] = from_f<bf16>(v);
  }
}

// The entry of a chunk: the last whose first chunk is at or before it.
__device__ __forceinline__ int entry_of(const Table& t, uint32_t chunk) {
  int lo = 0, hi = t.entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Sum of v over the block, on thread 0.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < kThreads / 32; ++i) v += part[i];
  return v;
}

// sums[chunk] = the chunk's sum of squares, in float64.
__global__ void __launch_bounds__(kThreads)
    square_sum_kernel(const __grid_constant__ Table t, double* sums) {
  const Entry& e = t.e[entry_of(t, blockIdx.x)];
  const int64_t i0 = (int64_t)(blockIdx.x - e.first_chunk) * kChunk;
  const int64_t i1 = min(e.count, i0 + kChunk);
  double s = 0;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
    const double v = load_as_float(e, i);
    s += v * v;
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// norm and the scale, from all chunks' sums.
__global__ void __launch_bounds__(kThreads)
    norm_kernel(const double* sums, int64_t chunks, double max_norm, float* norm, float* scale) {
  double s = 0;
  for (int64_t i = threadIdx.x; i < chunks; i += kThreads) s += sums[i];
  s = block_sum(s);
  if (threadIdx.x == 0) {
    const double n = sqrt(s);
    *norm = (float)n;
    *scale = isfinite(n) && n > max_norm ? (float)(max_norm / n) : 1.f;
  }
}

__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table t, const float* scale) {
  const Entry& e = t.e[entry_of(t, blockIdx.x)];
  const float f = *scale;
  if (f == 1.f && e.in == e.out) return;
  const int64_t i0 = (int64_t)(blockIdx.x - e.first_chunk) * kChunk;
  const int64_t i1 = min(e.count, i0 + kChunk);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
    store_from_float(e, i, load_as_float(e, i) * f);
}

xvec_gpu_status clip(const xvec_gpu_tensor* tensors, int num, double max_norm, float* d_norm,
                     cudaStream_t s) {
  int64_t chunks = 0;
  for (int i = 0; i < num; ++i) chunks += (tensors[i].count + kChunk - 1) / kChunk;
  Scratch sums, scale;
  xvec_gpu_status st;
  if ((st = sums.alloc((size_t)chunks * 8, s)) || (st = scale.alloc(4, s))) return st;
  Table t;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t done = 0;
    for (int i = 0; i < num;) {
      t.entries = 0;
      t.chunks = 0;
      for (; i < num && t.entries < kMaxEntries; ++i) {
        const int64_t c = (tensors[i].count + kChunk - 1) / kChunk;
        if (c == 0) continue;
        if (t.chunks + c > 0x7fffffff) break;
        t.e[t.entries++] = {tensors[i].in, tensors[i].out, tensors[i].count, tensors[i].storage,
                            t.chunks};
        t.chunks += (uint32_t)c;
      }
      if (t.entries == 0) continue;
      if (pass == 0)
        square_sum_kernel<<<t.chunks, kThreads, 0, s>>>(t, sums.as<double>() + done);
      else
        scale_kernel<<<t.chunks, kThreads, 0, s>>>(t, scale.as<float>());
      XVEC_LAUNCHED();
      XVEC_CUDA(cudaGetLastError());
      done += t.chunks;
    }
    if (pass == 0) {
      norm_kernel<<<1, kThreads, 0, s>>>(sums.as<double>(), chunks, max_norm, d_norm,
                                         scale.as<float>());
      XVEC_LAUNCHED();
      XVEC_CUDA(cudaGetLastError());
    }
  }
  return XVEC_GPU_OK;
}

// Whether an output overlaps another output or an input (an in-place tensor is
// one output): the byte ranges sorted by their start, each against the
// furthest end before it.  Inputs may overlap one another.
struct Range {
  uintptr_t begin, end;
  bool out;
};
bool overlapping(Range* r, int n) {
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t end_any = 0, end_out = 0;
  for (int i = 0; i < n; ++i) {
    if (r[i].begin < (r[i].out ? end_any : end_out)) return true;
    end_any = std::max(end_any, r[i].end);
    if (r[i].out) end_out = std::max(end_out, r[i].end);
  }
  return false;
}

}  // namespace
}  // namespace adapter
}  // namespace xvec

using namespace xvec;
using namespace xvec::adapter;

extern "C" xvec_gpu_status xvec_gpu_clip_gradients_device(int32_t device,
                                                          const xvec_gpu_tensor* tensors,
                                                          int32_t num_tensors, double max_norm,
                                                          float* d_norm, void* stream) {
  auto invalid = [](const char* what) {
    set_error("clip: %s", what);
    return XVEC_GPU_INVALID_ARGUMENT;
  };
  if (num_tensors < 0 || (num_tensors > 0 && !tensors)) return invalid("nil tensors");
  if (!d_norm || (uintptr_t)d_norm % 4) return invalid("the norm needs an aligned float32");
  if (!(max_norm >= 0)) return invalid("max_norm must be at least 0");
  for (int i = 0; i < num_tensors; ++i) {
    const xvec_gpu_tensor& t = tensors[i];
    if (t.storage != XVEC_STORAGE_FP32 && t.storage != XVEC_STORAGE_FP16 &&
        t.storage != XVEC_STORAGE_BF16)
      return invalid("invalid storage");
    const size_t size = t.storage == XVEC_STORAGE_FP32 ? 4 : 2;
    if (t.reserved != 0) return invalid("reserved must be 0");
    if (t.count < 0 || t.count > ((int64_t)1 << 40)) return invalid("invalid element count");
    if (t.count && (!t.in || !t.out)) return invalid("nil tensor");
    if ((uintptr_t)t.in % size || (uintptr_t)t.out % size)
      return invalid("a tensor is not aligned to its elements");
  }
  Range* ranges = new (std::nothrow) Range[2 * (size_t)num_tensors + 1];
  if (!ranges) return set_error("out of host memory"), XVEC_GPU_OUT_OF_MEMORY;
  int num = 0;
  ranges[num++] = {(uintptr_t)d_norm, (uintptr_t)d_norm + 4, true};
  for (int i = 0; i < num_tensors; ++i) {
    const xvec_gpu_tensor& t = tensors[i];
    if (t.count == 0) continue;
    const uintptr_t bytes = t.count * (t.storage == XVEC_STORAGE_FP32 ? 4 : 2);
    ranges[num++] = {(uintptr_t)t.out, (uintptr_t)t.out + bytes, true};
    if (t.in != t.out) ranges[num++] = {(uintptr_t)t.in, (uintptr_t)t.in + bytes, false};
  }
  const bool bad = overlapping(ranges, num);
  delete[] ranges;
  if (bad) return invalid("an output overlaps another tensor");
  DeviceGuard guard;
  if (xvec_gpu_status st = guard.set(device)) return st;
  return clip(tensors, num_tensors, max_norm, d_norm, static_cast<cudaStream_t>(stream));
}
