// clip.cu — the global norm of many gradient tensors and their clipping to it.
//
//   norm = sqrt(sum over all tensors of x^2),  out = x min(1, max_norm / norm)
//
// Two launches, both bound by memory.  The tensors are cut into chunks of 32 KB;
// block b takes chunks b, b + blocks, ...: the first launch leaves one float64 sum
// of squares per block, the second adds them (every block for itself, which
// saves a launch) and scales, its chunks in the opposite order, so that the
// last ones that the first launch read still lie in L2.  Which block adds
// what depends on the sizes alone, so results repeat.
//
// Squares: a 16-byte vector's are summed in float32 and added up in float64; a
// vector whose sum leaves float32's comfortable range (values around 1e-19 or
// 1e19, and what is not finite) is squared in float64, so that neither overflow
// nor underflow of a square matters.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <new>

#include "adapter.cuh"

namespace xvec {
namespace adapter {
namespace {

constexpr int kChunkBytes = 32768;
constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 6;

struct Entry {
  const void* in;
  void* out;
  int64_t count;
  int32_t storage;
  uint32_t first_chunk;  // of this launch
};
// Travels as a kernel parameter; three sizes, since a launch pays for its bytes (34
// tensors: 64 us in the largest, 32 in the middle one).
template <int N>
struct Table {
  int entries;
  uint32_t chunks;
  Entry e[N];
};
constexpr int kFew = 24, kSome = 120, kMany = 500;

__host__ __device__ constexpr int chunk_elems(int storage) {
  return storage == XVEC_STORAGE_FP32 ? kChunkBytes / 4 : kChunkBytes / 2;
}

// The entry of a chunk: the last whose first chunk is at or before it.
template <int N>
__device__ __forceinline__ int entry_of(const Table<N>& t, uint32_t chunk) {
  int lo = 0, hi = t.entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Sum of v over the block in a fixed order, on every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v += part[i];
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(T); ++j) v[j] = to_f(t[j]);
}

// Sum of the squares of one 16-byte vector.
template <typename T>
__device__ __forceinline__ double vector_squares(const uint4& u) {
  constexpr int N = 16 / sizeof(T);
  float v[N];
  unpack<T>(u, v);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) s = fmaf(v[j], v[j], s);
  if constexpr (!std::is_same<T, __half>::value) {
    if (!(s >= 1e-30f && s <= 1e37f)) {
      double d = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) d = fma((double)v[j], (double)v[j], d);
      return d;
    }
  }
  return s;
}

// Elements [i0, i1) of a tensor: the vectors between 16-byte boundaries, and
// the few elements before and after them one by one.
template <typename T>
__device__ __forceinline__ double square_range(const T* in, int64_t i0, int64_t i1) {
  constexpr int N = 16 / sizeof(T);
  const int64_t head = min(i1, i0 + (int64_t)((16 - (uintptr_t)(in + i0) % 16) % 16 / sizeof(T)));
  const int vectors = (int)((i1 - head) / N);
  const uint4* p = reinterpret_cast<const uint4*>(in + head);
  double s0 = 0, s1 = 0;
  int i = threadIdx.x;
  for (; i + 3 * kThreads < vectors; i += 4 * kThreads) {
    const uint4 a = p[i], b = p[i + kThreads], c = p[i + 2 * kThreads], d = p[i + 3 * kThreads];
    s0 += vector_squares<T>(a);
    s1 += vector_squares<T>(b);
    s0 += vector_squares<T>(c);
    s1 += vector_squares<T>(d);
  }
  for (; i < vectors; i += kThreads) s0 += vector_squares<T>(p[i]);
  const int64_t tail = head + (int64_t)vectors * N;
  const int64_t e = threadIdx.x < head - i0 ? i0 + threadIdx.x : tail + threadIdx.x - (head - i0);
  if (e < i1) {
    const double v = to_f(in[e]);
    s1 = fma(v, v, s1);
  }
  return s0 + s1;
}

template <typename T>
__device__ __forceinline__ uint4 scaled(const uint4& u, float f) {
  constexpr int N = 16 / sizeof(T);
  float v[N];
  unpack<T>(u, v);
  uint4 r;
  T* t = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = from_f<T>(v[j] * f);
  return r;
}

template <typename T>
__device__ __forceinline__ void scale_range(const T* in, T* out, int64_t i0, int64_t i1, float f) {
  constexpr int N = 16 / sizeof(T);
  // No common 16-byte boundaries: one by one (260M float32 values 846 us, else 511).
  if (((uintptr_t)in ^ (uintptr_t)out) % 16) {
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) out[i] = from_f<T>(to_f(in[i]) * f);
    return;
  }
  const int64_t head = min(i1, i0 + (int64_t)((16 - (uintptr_t)(in + i0) % 16) % 16 / sizeof(T)));
  const int vectors = (int)((i1 - head) / N);
  const uint4* p = reinterpret_cast<const uint4*>(in + head);
  uint4* q = reinterpret_cast<uint4*>(out + head);
  int i = threadIdx.x;
  for (; i + 3 * kThreads < vectors; i += 4 * kThreads) {
    const uint4 a = p[i], b = p[i + kThreads], c = p[i + 2 * kThreads], d = p[i + 3 * kThreads];
    q[i] = scaled<T>(a, f);
    q[i + kThreads] = scaled<T>(b, f);
    q[i + 2 * kThreads] = scaled<T>(c, f);
    q[i + 3 * kThreads] = scaled<T>(d, f);
  }
  for (; i < vectors; i += kThreads) q[i] = scaled<T>(p[i], f);
  const int64_t tail = head + (int64_t)vectors * N;
  const int64_t e = threadIdx.x < head - i0 ? i0 + threadIdx.x : tail + threadIdx.x - (head - i0);
  if (e < i1) out[e] = from_f<T>(to_f(in[e]) * f);
}

// The same by a factor that float32 cannot hold to its full precision.
template <typename T>
__device__ __noinline__ void scale_range_tiny(const T* in, T* out, int64_t i0, int64_t i1,
                                              double f) {
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads)
    out[i] = from_f<T>((float)(to_f(in[i]) * f));
}

// sums[block] = the sum of squares of the block's chunks.
template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    square_sum_kernel(const __grid_constant__ Table<N> t, double* sums) {
  pdl_begin();
  double s = 0;
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = t.e[entry_of(t, c)];
    const int64_t i0 = (int64_t)(c - e.first_chunk) * chunk_elems(e.storage);
    const int64_t i1 = min(e.count, i0 + chunk_elems(e.storage));
    if (e.storage == XVEC_STORAGE_FP32)
      s += square_range(static_cast<const float*>(e.in), i0, i1);
    else if (e.storage == XVEC_STORAGE_FP16)
      s += square_range(static_cast<const __half*>(e.in), i0, i1);
    else
      s += square_range(static_cast<const bf16*>(e.in), i0, i1);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    scale_kernel(const __grid_constant__ Table<N> t, const double* sums, int num_sums,
                 double max_norm, float* norm) {
  pdl_begin();
  double s = 0;
  for (int i = threadIdx.x; i < num_sums; i += kThreads) s += sums[i];
  const double n = sqrt(block_sum(s));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double factor = isfinite(n) && n > max_norm ? max_norm / n : 1.0;
  const float f = (float)factor;
  // Below float32's normal numbers the factor loses bits, down to zero, while its
  // product with gradients near 1e38 is an ordinary number: float64 there, and
  // nothing to gain from speed.  (float16 values times such a factor are zeros.)
  const bool tiny = factor > 0 && factor < FLT_MIN;
  if (blockIdx.x >= t.chunks) return;
  for (uint32_t c = blockIdx.x + (t.chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x;;
       c -= gridDim.x) {
    const Entry& e = t.e[entry_of(t, c)];
    if (f != 1.f || e.in != e.out) {
      const int64_t i0 = (int64_t)(c - e.first_chunk) * chunk_elems(e.storage);
      const int64_t i1 = min(e.count, i0 + chunk_elems(e.storage));
      if (tiny && e.storage == XVEC_STORAGE_FP32)
        scale_range_tiny(static_cast<const float*>(e.in), static_cast<float*>(e.out), i0, i1,
                         factor);
      else if (tiny && e.storage == XVEC_STORAGE_BF16)
        scale_range_tiny(static_cast<const bf16*>(e.in), static_cast<bf16*>(e.out), i0, i1, factor);
      else if (e.storage == XVEC_STORAGE_FP32)
        scale_range(static_cast<const float*>(e.in), static_cast<float*>(e.out), i0, i1, f);
      else if (e.storage == XVEC_STORAGE_FP16)
        scale_range(static_cast<const __half*>(e.in), static_cast<__half*>(e.out), i0, i1, f);
      else
        scale_range(static_cast<const bf16*>(e.in), static_cast<bf16*>(e.out), i0, i1, f);
    }
    if (c < gridDim.x) break;
  }
}

// Launches over all tensors, N at a time: sums (pass 0) and scaling (pass 1).
template <int N>
xvec_gpu_status clip(const xvec_gpu_tensor* tensors, int num, double max_norm, float* d_norm,
                     int sms, const DeviceGuard& guard, cudaStream_t s) {
  const int max_blocks = sms * kBlocksPerSm;
  Table<N> t;
  // Fills t from tensor *i on; false when nothing is left.
  auto fill = [&](int* i) {
    t.entries = 0;
    t.chunks = 0;
    for (; *i < num && t.entries < N; ++*i) {
      const xvec_gpu_tensor& x = tensors[*i];
      const int64_t c = (x.count + chunk_elems(x.storage) - 1) / chunk_elems(x.storage);
      if (c == 0) continue;
      if (t.chunks + c > 0x7fffffff) break;
      t.e[t.entries++] = {x.in, x.out, x.count, x.storage, t.chunks};
      t.chunks += (uint32_t)c;
    }
    return t.entries > 0;
  };
  int blocks = 0;
  for (int i = 0; fill(&i);) blocks += (int)std::min<uint32_t>(t.chunks, max_blocks);
  Scratch sums;
  if (xvec_gpu_status st = sums.alloc((size_t)blocks * 8, s, guard.pool)) return st;
  int done = 0;
  for (int i = 0; fill(&i);) {
    const int b = (int)std::min<uint32_t>(t.chunks, max_blocks);
    XVEC_CUDA(launch_pdl(square_sum_kernel<N>, dim3(b), kThreads, 0, s, 1, t,
                         sums.as<double>() + done));
    done += b;
  }
  int i = 0;
  for (int pass = 0; fill(&i) || pass == 0; ++pass) {
    const int b = std::max(1, (int)std::min<uint32_t>(t.chunks, max_blocks));
    XVEC_CUDA(launch_pdl(scale_kernel<N>, dim3(b), kThreads, 0, s, 1, t, sums.as<double>(), blocks,
                         max_norm, pass == 0 ? d_norm : nullptr));
    if (t.entries == 0) break;
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
  int sms = 0;
  if (xvec_gpu_status st = count_sms(device, &sms)) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return num_tensors <= kFew    ? clip<kFew>(tensors, num_tensors, max_norm, d_norm, sms, guard, s)
         : num_tensors <= kSome ? clip<kSome>(tensors, num_tensors, max_norm, d_norm, sms, guard, s)
                                : clip<kMany>(tensors, num_tensors, max_norm, d_norm, sms, guard, s);
}
