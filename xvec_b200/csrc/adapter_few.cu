// adapter_few.cu — the adapter's forward calls for a few rows (queries).
//
// With so few rows every weight is used a few times only: bound by reading the
// weights once, and at the smallest sizes by latency.  A block owns kCols output
// columns for up to eight rows; its four warps split the depth (blocks of 256, 8
// elements a lane), so that even a small layer has its weights under way on every
// SM at once, and the x rows come from L1 or L2.  float32 multiply-adds; the partial
// sums of all rows and columns are added across the lanes in a halving exchange
// that leaves each sum on one lane, then over the warps in shared memory, in a
// fixed order.  More columns a block use an x row more often; fewer spread a small
// weight over more SMs: one or two columns up to four rows, four for eight.  More than
// eight rows read the weights again for each eight.
#include "adapter.cuh"

namespace xvec {
namespace adapter {
namespace {

constexpr int kWarps = 4;

// v[0..N) of every lane added over the warp; sum i ends in v[0] of the lanes whose
// leading bits (the first log2 N of 5) are i.
template <int N>
__device__ __forceinline__ float scatter_sum(float (&v)[N], int lane) {
  static_assert(N <= 32 && (N & (N - 1)) == 0, "a power of two up to the warp");
  int width = N;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (width > 1) {
      width >>= 1;
      const bool high = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < width) {
          const float send = high ? v[i] : v[i + width];
          const float keep = high ? v[i + width] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}
constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// VEC: x and the weights allow 16-byte accesses, in_dim is a multiple of 8.
template <typename T, bool GATED, int ROWS, int COLS, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) few_rows_kernel(const __grid_constant__ FewRows p) {
  constexpr int W = GATED ? 2 : 1;
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * COLS, r0 = blockIdx.y * ROWS;
  const T* x = static_cast<const T*>(p.x);
  float sum[W][ROWS * COLS] = {};
#pragma unroll 2
  for (int k = threadIdx.x * 8; k < p.in_dim; k += kWarps * 256) {
    const int count = p.in_dim - k;
    Eight<T, VEC> w[W][COLS];
#pragma unroll
    for (int m = 0; m < W; ++m)
#pragma unroll
      for (int c = 0; c < COLS; ++c)  // (a column that does not exist repeats the last)
        w[m][c].load(
            static_cast<const T*>(p.w[m]) + (int64_t)min(c0 + c, p.out_dim - 1) * p.ldw + k, count);
#pragma unroll
    for (int m = 0; m < W; ++m)
#pragma unroll
      for (int c = 0; c < COLS; ++c) w[m][c].settle();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      Eight<T, VEC> v;
      v.load(x + (int64_t)min(r0 + r, p.n - 1) * p.ldx + k, count);
      v.settle();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = VEC || j < count;  // (past the row's end lie other elements)
#pragma unroll
        for (int m = 0; m < W; ++m)
#pragma unroll
          for (int c = 0; c < COLS; ++c)
            sum[m][r * COLS + c] =
                fmaf(in ? v[j] : 0.f, in ? w[m][c][j] : 0.f, sum[m][r * COLS + c]);
      }
    }
  }
  // Lane `lane` >> kShift holds one sum of its warp; the first warp adds them up.
  constexpr int kSums = ROWS * COLS, kShift = 5 - log2_of(kSums);
  __shared__ float part[W][kWarps][kSums];
#pragma unroll
  for (int m = 0; m < W; ++m) {
    const float total = scatter_sum(sum[m], lane);
    if ((lane & ((1 << kShift) - 1)) == 0) part[m][warp][lane >> kShift] = total;
  }
  __syncthreads();
  const int r = r0 + (int)threadIdx.x / COLS, c = c0 + (int)threadIdx.x % COLS;
  if (threadIdx.x >= kSums || r >= p.n || c >= p.out_dim) return;
  float pre[W];
#pragma unroll
  for (int m = 0; m < W; ++m) {
    pre[m] = part[m][0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) pre[m] += part[m][w][threadIdx.x];
    if (p.bias[m]) pre[m] += to_f(static_cast<const T*>(p.bias[m])[c]);
    if (p.save[m]) static_cast<T*>(p.save[m])[r * p.lds + c] = from_f<T>(pre[m]);
  }
  float y = activate<T>(p.act, pre[0]);
  if (GATED) y *= pre[W - 1];
  if (!GATED && p.residual) y += to_f(static_cast<const T*>(p.residual)[r * p.ldr + c]);
  static_cast<T*>(p.out)[r * p.ldo + c] = from_f<T>(y);
}

template <typename T, bool GATED, int ROWS, int COLS>
xvec_gpu_status launch(const FewRows& f, cudaStream_t s) {
  const bool vec = aligned16(f.x, f.ldx, sizeof(T)) && aligned16(f.w[0], f.ldw, sizeof(T)) &&
                   aligned16(f.w[1], f.ldw, sizeof(T)) && f.in_dim % 8 == 0;
  auto* kern = vec ? few_rows_kernel<T, GATED, ROWS, COLS, true>
                   : few_rows_kernel<T, GATED, ROWS, COLS, false>;
  XVEC_CUDA(launch_pdl(kern, dim3((f.out_dim + COLS - 1) / COLS, (f.n + ROWS - 1) / ROWS),
                       kWarps * 32, 0, s, 1, f));
  return XVEC_GPU_OK;
}

template <typename T, bool GATED>
xvec_gpu_status by_rows(const FewRows& f, cudaStream_t s) {
  if (f.n == 1) return launch<T, GATED, 1, 1>(f, s);
  if (f.n == 2) return launch<T, GATED, 2, 1>(f, s);
  if (f.n <= 4) return launch<T, GATED, 4, GATED ? 1 : 2>(f, s);
  return launch<T, GATED, 8, GATED ? 2 : 4>(f, s);
}
template <typename T>
xvec_gpu_status by_kind(const FewRows& f, cudaStream_t s) {
  return f.w[1] ? by_rows<T, true>(f, s) : by_rows<T, false>(f, s);
}

}  // namespace

xvec_gpu_status few_rows(int storage, const FewRows& f, cudaStream_t s) {
  return storage == XVEC_STORAGE_FP32   ? by_kind<float>(f, s)
         : storage == XVEC_STORAGE_FP16 ? by_kind<__half>(f, s)
                                        : by_kind<bf16>(f, s);
}

}  // namespace adapter
}  // namespace xvec
