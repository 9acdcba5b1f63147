// adapter.cu — the learned adapter: an affine layer, a gated block and their
// gradients, on device memory and the caller's stream.
//
//   linear:   z = x W' + b,  y = act(z) + r
//   gated:    g = x Wg' + bg,  u = x Wu' + bu,  h = act(g) u
//   backward: dz = dy act'(z)  |  dg = dh u act'(g), du = dh act(g)
//             dx = dz W        |  dx = dg Wg + du Wu
//             dW = dz' x, db = column sums of dz (likewise for g and u)
//
// The entry points check their arguments, put the pre-activation gradients
// (elementwise, with their column sums) into scratch and run the products.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "adapter.cuh"

namespace xvec {
namespace adapter {
namespace {

constexpr int64_t kMaxDim = 1 << 20;
constexpr int kMaxDevices = 64;

// --- products: one 64 x 64 tile per block, float32 sums in registers ------
constexpr int kTile = 64, kDepth = 16;

template <typename T>
struct Operand {
  const T* p[2];
  int64_t outer, inner;  // strides of the row (or column) index and of the depth index
};

template <typename T, int MODE>
__global__ void __launch_bounds__(256)
    product_kernel(Product p, Operand<T> a, Operand<T> b, int z_parts) {
  __shared__ float as[kDepth][kTile + 1], bs[2][kDepth][kTile + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t r0 = (int64_t)blockIdx.x * kTile, c0 = (int64_t)blockIdx.y * kTile;
  const int z = blockIdx.z;
  constexpr int kSums = MODE == kGated ? 2 : 1;
  // Two levels of sums (every 256 terms), so that long ones keep float32 accuracy.
  float acc[kSums][4][4] = {}, total[kSums][4][4] = {};
  for (int seg = 0; seg < z_parts; ++seg) {
    const T* ap = a.p[MODE == kDw ? z : MODE == kDx ? seg : 0];
    for (int64_t k0 = 0; k0 < p.depth; k0 += kDepth) {
      for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
        // The faster index follows the operand's contiguous direction.
        const int kk = a.inner == 1 ? i % kDepth : i / kTile;
        const int rr = a.inner == 1 ? i / kDepth : i % kTile;
        const bool in = r0 + rr < p.rows && k0 + kk < p.depth;
        as[kk][rr] = in ? to_f(ap[(r0 + rr) * a.outer + (k0 + kk) * a.inner]) : 0.f;
      }
      for (int s = 0; s < kSums; ++s) {
        const T* bp = b.p[MODE == kGated ? s : MODE == kDx ? seg : 0];
        for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
          const int kk = b.inner == 1 ? i % kDepth : i / kTile;
          const int cc = b.inner == 1 ? i / kDepth : i % kTile;
          const bool in = c0 + cc < p.cols && k0 + kk < p.depth;
          bs[s][kk][cc] = in ? to_f(bp[(c0 + cc) * b.outer + (k0 + kk) * b.inner]) : 0.f;
        }
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kDepth; ++kk)
#pragma unroll
        for (int s = 0; s < kSums; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[s][i][j] = fmaf(as[kk][ty + 16 * i], bs[s][kk][tx + 16 * j], acc[s][i][j]);
      __syncthreads();
      if (k0 % 256 == 256 - kDepth || k0 + kDepth >= p.depth)
#pragma unroll
        for (int s = 0; s < kSums; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) total[s][i][j] += acc[s][i][j], acc[s][i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + ty + 16 * i, c = c0 + tx + 16 * j;
      if (r >= p.rows || c >= p.cols) continue;
      float v = total[0][i][j];
      if (MODE == kLinear || MODE == kGated) {
        if (p.bias[0]) v += to_f(static_cast<const T*>(p.bias[0])[c]);
        if (p.save[0]) static_cast<T*>(p.save[0])[r * p.lds + c] = from_f<T>(v);
        v = activate(p.act, v);
      }
      if constexpr (MODE == kGated) {
        float u = total[1][i][j];
        if (p.bias[1]) u += to_f(static_cast<const T*>(p.bias[1])[c]);
        if (p.save[1]) static_cast<T*>(p.save[1])[r * p.lds + c] = from_f<T>(u);
        v *= u;
      }
      if (MODE == kLinear && p.residual)
        v += to_f(static_cast<const T*>(p.residual)[r * p.ldr + c]);
      static_cast<T*>(p.out[MODE == kDw ? z : 0])[r * p.ldo + c] = from_f<T>(v);
    }
}

template <typename T, int MODE>
xvec_gpu_status launch_product(const Product& p, cudaStream_t s) {
  Operand<T> a{{static_cast<const T*>(p.a[0]), static_cast<const T*>(p.a[1])}, p.lda, 1};
  Operand<T> b{{static_cast<const T*>(p.b[0]), static_cast<const T*>(p.b[1])}, p.ldb, 1};
  if (MODE == kDw) std::swap(a.outer, a.inner);
  if (MODE == kDw || MODE == kDx) std::swap(b.outer, b.inner);
  const dim3 grid((unsigned)((p.rows + kTile - 1) / kTile), (unsigned)((p.cols + kTile - 1) / kTile),
                  MODE == kDw ? p.parts : 1);
  product_kernel<T, MODE><<<grid, 256, 0, s>>>(p, a, b, MODE == kDx ? p.parts : 1);
  XVEC_LAUNCHED();
  XVEC_CUDA(cudaGetLastError());
  return XVEC_GPU_OK;
}

template <typename T>
xvec_gpu_status run_product_t(const Product& p, cudaStream_t s) {
  switch (p.mode) {
    case kLinear: return launch_product<T, kLinear>(p, s);
    case kGated: return launch_product<T, kGated>(p, s);
    case kDx: return launch_product<T, kDx>(p, s);
    default: return launch_product<T, kDw>(p, s);
  }
}

xvec_gpu_status run_product(const Product& p, cudaStream_t s) {
  if (p.rows == 0 || p.cols == 0) return XVEC_GPU_OK;
  switch (p.storage) {
    case XVEC_STORAGE_FP32: return run_product_t<float>(p, s);
    case XVEC_STORAGE_FP16: return run_product_t<__half>(p, s);
    default: return run_product_t<bf16>(p, s);
  }
}

// --- pre-activation gradients and their column sums -----------------------
// dz = dy act'(z), or (GATED) dg = dh u act'(g) and du = dh act(g), rounded to
// T; partial [2][chunks][m]: the column sums of each row chunk in float32,
// before the rounding.
template <typename T, bool GATED>
__global__ void __launch_bounds__(256)
    slope_kernel(const T* dy, int64_t lddy, const T* z, const T* u, int64_t ldz, int64_t n, int m,
                 int act, int64_t rows_per_chunk, T* out0, T* out1, float* partial) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= m) return;
  const int64_t r0 = blockIdx.y * rows_per_chunk;
  const int64_t r1 = min(n, r0 + rows_per_chunk);
  float s0 = 0.f, s1 = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float d = to_f(dy[r * lddy + c]);
    if (GATED) {
      const float g = to_f(z[r * ldz + c]), v = to_f(u[r * ldz + c]);
      const float dg = d * v * slope(act, g), du = d * activate(act, g);
      out0[r * m + c] = from_f<T>(dg);
      out1[r * m + c] = from_f<T>(du);
      s0 += dg;
      s1 += du;
    } else {
      const float v = act == XVEC_ACT_NONE ? d : d * slope(act, to_f(z[r * ldz + c]));
      out0[r * m + c] = from_f<T>(v);
      s0 += v;
    }
  }
  if (partial) {
    partial[(int64_t)blockIdx.y * m + c] = s0;
    if (GATED) partial[((int64_t)gridDim.y + blockIdx.y) * m + c] = s1;
  }
}

// out[c] = the sum over the chunks, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
    column_sum_kernel(const float* partial, int chunks, int m, T* out0, T* out1) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  T* out = blockIdx.y ? out1 : out0;
  if (c >= m || !out) return;
  const float* p = partial + (int64_t)blockIdx.y * chunks * m + c;
  double s = 0;
  for (int i = 0; i < chunks; ++i) s += p[(int64_t)i * m];
  out[c] = from_f<T>((float)s);
}

template <typename T>
xvec_gpu_status slopes_t(const void* dy, int64_t lddy, const void* z, const void* u, int64_t ldz,
                         int64_t n, int m, int act, void* out0, void* out1, void* db0, void* db1,
                         cudaStream_t s) {
  const int chunks = (int)std::max<int64_t>(1, std::min<int64_t>(64, (n + 31) / 32));
  const int64_t per = (n + chunks - 1) / chunks;
  Scratch partial;
  xvec_gpu_status st;
  if (db0 || db1)
    if ((st = partial.alloc((size_t)2 * chunks * m * 4, s))) return st;
  const dim3 grid((m + 255) / 256, chunks);
  auto* kern = u ? slope_kernel<T, true> : slope_kernel<T, false>;
  kern<<<grid, 256, 0, s>>>(static_cast<const T*>(dy), lddy, static_cast<const T*>(z),
                            static_cast<const T*>(u), ldz, n, m, act, per,
                            static_cast<T*>(out0), static_cast<T*>(out1), partial.as<float>());
  XVEC_LAUNCHED();
  XVEC_CUDA(cudaGetLastError());
  if (db0 || db1) {
    column_sum_kernel<T><<<dim3((m + 255) / 256, 2), 256, 0, s>>>(
        partial.as<float>(), chunks, m, static_cast<T*>(db0), static_cast<T*>(db1));
    XVEC_LAUNCHED();
    XVEC_CUDA(cudaGetLastError());
  }
  return XVEC_GPU_OK;
}

xvec_gpu_status slopes(int storage, const void* dy, int64_t lddy, const void* z, const void* u,
                       int64_t ldz, int64_t n, int m, int act, void* out0, void* out1, void* db0,
                       void* db1, cudaStream_t s) {
  auto* f = storage == XVEC_STORAGE_FP32   ? slopes_t<float>
            : storage == XVEC_STORAGE_FP16 ? slopes_t<__half>
                                           : slopes_t<bf16>;
  return f(dy, lddy, z, u, ldz, n, m, act, out0, out1, db0, db1, s);
}

// --- argument checks --------------------------------------------------------
size_t elem_bytes(int storage) { return storage == XVEC_STORAGE_FP32 ? 4 : 2; }

xvec_gpu_status invalid(const char* what) {
  set_error("adapter: %s", what);
  return XVEC_GPU_INVALID_ARGUMENT;
}

struct Matrix {
  const char* name;
  const void* p;
  int64_t rows, cols, ld;
};

// Whether two matrices of one element size share an element.  Column ranges
// of one wider matrix (equal leading dimensions) may interleave.
bool share(const Matrix& a, const Matrix& b, size_t size) {
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
  const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
  const uintptr_t a1 = a0 + ((uint64_t)(a.rows - 1) * a.ld + a.cols) * size;
  const uintptr_t b1 = b0 + ((uint64_t)(b.rows - 1) * b.ld + b.cols) * size;
  if (a1 <= b0 || b1 <= a0) return false;
  const bool strided_a = a.rows > 1, strided_b = b.rows > 1;
  if (strided_a && strided_b && a.ld != b.ld) return true;
  if (!strided_a && !strided_b) return true;
  const int64_t ld = strided_a ? a.ld : b.ld;
  const int64_t off = (int64_t)(b0 - a0);  // bytes, either sign
  const int64_t pitch = ld * (int64_t)size;
  if (a.cols > ld || b.cols > ld) return true;
  const int64_t d = ((off % pitch) + pitch) % pitch;
  return d < a.cols * (int64_t)size || d + b.cols * (int64_t)size > pitch;
}

// Fills in contiguous leading dimensions and checks one call's matrices.
struct Check {
  size_t size;
  Matrix ins[8], outs[6];  // a call has at most 6 of either
  int num_ins = 0, num_outs = 0;
  xvec_gpu_status st = XVEC_GPU_OK;
  explicit Check(size_t size) : size(size) {}

  void ld(const char* name, const void* p, int64_t cols, int64_t* ld) {
    if (st || !p) return;
    if (*ld == 0) *ld = cols;
    if (*ld < cols) {
      set_error("adapter: leading dimension %lld of %s is less than its %lld columns",
                (long long)*ld, name, (long long)cols);
      st = XVEC_GPU_INVALID_ARGUMENT;
    } else if (*ld > ((int64_t)1 << 27)) {
      set_error("adapter: leading dimension %lld of %s is too large", (long long)*ld, name);
      st = XVEC_GPU_INVALID_ARGUMENT;
    }
  }
  void in(const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld) {
    aligned(name, p);
    ins[num_ins++] = {name, p, rows, cols, ld};
  }
  void out(const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld) {
    aligned(name, p);
    outs[num_outs++] = {name, p, rows, cols, ld};
  }
  void aligned(const char* name, const void* p) {
    if (st || (uintptr_t)p % size == 0) return;
    set_error("adapter: %s is not aligned to its elements", name);
    st = XVEC_GPU_INVALID_ARGUMENT;
  }
  // `same_ok`: an output that may be the input `same` itself.
  xvec_gpu_status overlaps(const char* same_out = nullptr, const char* same_in = nullptr) {
    if (st) return st;
    for (int i = 0; i < num_outs; ++i) {
      for (int j = 0; j < num_ins; ++j) {
        const Matrix& m = ins[j];
        const bool same = same_out && outs[i].name == same_out && m.name == same_in &&
                          outs[i].p == m.p && (outs[i].ld == m.ld || m.rows <= 1);
        if (!same && share(outs[i], m, size)) {
          set_error("adapter: %s overlaps %s", outs[i].name, m.name);
          return st = XVEC_GPU_INVALID_ARGUMENT;
        }
      }
      for (int j = i + 1; j < num_outs; ++j)
        if (share(outs[i], outs[j], size)) {
          set_error("adapter: %s overlaps %s", outs[i].name, outs[j].name);
          return st = XVEC_GPU_INVALID_ARGUMENT;
        }
    }
    return XVEC_GPU_OK;
  }
};

template <typename Args>
xvec_gpu_status check_shape(const Args* a) {
  if (!a) return invalid("nil arguments");
  if (a->storage != XVEC_STORAGE_FP32 && a->storage != XVEC_STORAGE_FP16 &&
      a->storage != XVEC_STORAGE_BF16)
    return invalid("invalid storage");
  if (a->activation < XVEC_ACT_NONE || a->activation > XVEC_ACT_SILU)
    return invalid("invalid activation");
  if (a->in_dim <= 0 || a->out_dim <= 0 || a->in_dim > kMaxDim || a->out_dim > kMaxDim)
    return invalid("dimensions must be in [1, 1048576]");
  if (a->n < 0 || a->n > INT_MAX - 1024) return invalid("row count must be in [0, 2^31 - 1025]");
  if (a->reserved != 0) return invalid("reserved must be 0");
  return XVEC_GPU_OK;
}

}  // namespace

xvec_gpu_status DeviceGuard::set(int device) {
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count) {
    cudaGetLastError();
    set_error("CUDA device %d is not available", device);
    return XVEC_GPU_UNSUPPORTED;
  }
  int now = 0;
  XVEC_CUDA(cudaGetDevice(&now));
  if (now != device) {
    XVEC_CUDA(cudaSetDevice(device));
    before = now;
  }
  static std::atomic<bool> ready[kMaxDevices];
  if (device < kMaxDevices && ready[device].load(std::memory_order_acquire)) return XVEC_GPU_OK;
  int major = 0, minor = 0;
  XVEC_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
  XVEC_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
  if (major != 10 || minor != 0) {
    set_error("device %d is not an sm_100 (B200) device", device);
    return XVEC_GPU_UNSUPPORTED;
  }
  // Keep freed stream-ordered scratch in the pool between calls (a setting
  // that a stream capture in progress would otherwise refuse).
  cudaMemPool_t pool;
  XVEC_CUDA(cudaDeviceGetDefaultMemPool(&pool, device));
  uint64_t threshold = UINT64_MAX;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  XVEC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  const cudaError_t set = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &threshold);
  XVEC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  XVEC_CUDA(set);
  if (device < kMaxDevices) ready[device].store(true, std::memory_order_release);
  return XVEC_GPU_OK;
}

}  // namespace adapter
}  // namespace xvec

using namespace xvec;
using namespace xvec::adapter;

extern "C" xvec_gpu_status xvec_gpu_linear_device(const xvec_gpu_linear_args* args) {
  xvec_gpu_status st = check_shape(args);
  if (st) return st;
  xvec_gpu_linear_args a = *args;
  if (!a.weight || (a.n && (!a.x || !a.y))) return invalid("x, weight and y are required");
  Check c(elem_bytes(a.storage));
  c.ld("x", a.x, a.in_dim, &a.ldx);
  c.ld("weight", a.weight, a.in_dim, &a.ldw);
  c.ld("residual", a.residual, a.out_dim, &a.ldr);
  c.ld("y", a.y, a.out_dim, &a.ldy);
  c.ld("preact", a.preact, a.out_dim, &a.ldz);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("weight", a.weight, a.out_dim, a.in_dim, a.ldw);
  c.in("bias", a.bias, 1, a.out_dim, a.out_dim);
  const char *y = "y", *residual = "residual";
  c.in(residual, a.residual, a.n, a.out_dim, a.ldr);
  c.out(y, a.y, a.n, a.out_dim, a.ldy);
  c.out("preact", a.preact, a.n, a.out_dim, a.ldz);
  if ((st = c.overlaps(y, residual))) return st;
  if (a.n == 0) return XVEC_GPU_OK;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  Product p;
  p.mode = kLinear;
  p.storage = a.storage;
  p.rows = a.n, p.cols = a.out_dim, p.depth = a.in_dim;
  p.a[0] = a.x, p.lda = a.ldx;
  p.b[0] = a.weight, p.ldb = a.ldw;
  p.bias[0] = a.bias;
  p.residual = a.residual, p.ldr = a.ldr;
  p.out[0] = a.y, p.ldo = a.ldy;
  p.save[0] = a.preact, p.lds = a.ldz;
  p.act = a.activation;
  return run_product(p, static_cast<cudaStream_t>(a.stream));
}

extern "C" xvec_gpu_status xvec_gpu_gated_device(const xvec_gpu_gated_args* args) {
  xvec_gpu_status st = check_shape(args);
  if (st) return st;
  xvec_gpu_gated_args a = *args;
  if (!a.gate_weight || !a.up_weight || (a.n && (!a.x || !a.h)))
    return invalid("x, gate_weight, up_weight and h are required");
  if (!a.gate != !a.up) return invalid("gate and up are given together or not at all");
  Check c(elem_bytes(a.storage));
  c.ld("x", a.x, a.in_dim, &a.ldx);
  c.ld("the weights", a.gate_weight, a.in_dim, &a.ldw);
  c.ld("h", a.h, a.out_dim, &a.ldh);
  c.ld("gate and up", a.gate, a.out_dim, &a.ldg);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("gate_weight", a.gate_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("up_weight", a.up_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("gate_bias", a.gate_bias, 1, a.out_dim, a.out_dim);
  c.in("up_bias", a.up_bias, 1, a.out_dim, a.out_dim);
  c.out("h", a.h, a.n, a.out_dim, a.ldh);
  c.out("gate", a.gate, a.n, a.out_dim, a.ldg);
  c.out("up", a.up, a.n, a.out_dim, a.ldg);
  if ((st = c.overlaps())) return st;
  if (a.n == 0) return XVEC_GPU_OK;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  Product p;
  p.mode = kGated;
  p.storage = a.storage;
  p.rows = a.n, p.cols = a.out_dim, p.depth = a.in_dim;
  p.a[0] = a.x, p.lda = a.ldx;
  p.b[0] = a.gate_weight, p.b[1] = a.up_weight, p.ldb = a.ldw;
  p.bias[0] = a.gate_bias, p.bias[1] = a.up_bias;
  p.out[0] = a.h, p.ldo = a.ldh;
  p.save[0] = a.gate, p.save[1] = a.up, p.lds = a.ldg;
  p.act = a.activation;
  return run_product(p, static_cast<cudaStream_t>(a.stream));
}

namespace xvec {
namespace adapter {
namespace {

// The backward pass of either block: `parts` 1 (linear) or 2 (gated).
struct Backward {
  int storage, act, parts;
  int64_t n;
  int in_dim, out_dim;
  const void *dy, *x, *w[2], *pre[2];
  void *dx, *dw[2], *db[2];
  int64_t lddy, ldx, ldw, ldpre, lddx, lddw;
  int32_t* status;
  cudaStream_t stream;
};

xvec_gpu_status run_backward(const Backward& b) {
  cudaStream_t s = b.stream;
  const size_t size = elem_bytes(b.storage);
  xvec_gpu_status st;
  const bool products = b.dx || b.dw[0] || b.dw[1];
  if (b.n == 0) {
    for (int i = 0; i < b.parts; ++i) {
      if (b.dw[i])
        XVEC_CUDA(cudaMemset2DAsync(b.dw[i], b.lddw * size, 0, b.in_dim * size, b.out_dim, s));
      if (b.db[i]) XVEC_CUDA(cudaMemsetAsync(b.db[i], 0, b.out_dim * size, s));
    }
    return XVEC_GPU_OK;
  }
  if (!products && !b.db[0] && !b.db[1]) return XVEC_GPU_OK;
  Scratch dz[2];
  for (int i = 0; i < b.parts; ++i)
    if ((st = dz[i].alloc((size_t)b.n * b.out_dim * size, s))) return st;
  if ((st = slopes(b.storage, b.dy, b.lddy, b.pre[0], b.parts == 2 ? b.pre[1] : nullptr, b.ldpre,
                   b.n, b.out_dim, b.act, dz[0].ptr, dz[1].ptr, b.db[0], b.db[1], s)))
    return st;
  if (b.dx) {
    Product p;
    p.mode = kDx;
    p.storage = b.storage;
    p.rows = b.n, p.cols = b.in_dim, p.depth = b.out_dim;
    p.parts = b.parts;
    for (int i = 0; i < b.parts; ++i) p.a[i] = dz[i].ptr, p.b[i] = b.w[i];
    p.lda = b.out_dim, p.ldb = b.ldw;
    p.out[0] = b.dx, p.ldo = b.lddx;
    if ((st = run_product(p, s))) return st;
  }
  if (b.dw[0] || b.dw[1]) {
    Product p;
    p.mode = kDw;
    p.storage = b.storage;
    p.rows = b.out_dim, p.cols = b.in_dim, p.depth = b.n;
    p.parts = 0;
    for (int i = 0; i < b.parts; ++i)
      if (b.dw[i]) p.a[p.parts] = dz[i].ptr, p.out[p.parts] = b.dw[i], ++p.parts;
    p.b[0] = b.x;
    p.lda = b.out_dim, p.ldb = b.ldx;
    p.ldo = b.lddw;
    if ((st = run_product(p, s))) return st;
  }
  return XVEC_GPU_OK;
}

}  // namespace
}  // namespace adapter
}  // namespace xvec

extern "C" xvec_gpu_status xvec_gpu_linear_backward_device(
    const xvec_gpu_linear_backward_args* args) {
  xvec_gpu_status st = check_shape(args);
  if (st) return st;
  xvec_gpu_linear_backward_args a = *args;
  if (a.n && !a.dy) return invalid("dy is required");
  if (a.dx && !a.weight) return invalid("dx needs weight");
  if (a.n && a.dweight && !a.x) return invalid("dweight needs x");
  if (a.n && a.activation != XVEC_ACT_NONE && !a.preact) return invalid("the activation needs preact");
  Check c(elem_bytes(a.storage));
  c.ld("dy", a.dy, a.out_dim, &a.lddy);
  c.ld("x", a.x, a.in_dim, &a.ldx);
  c.ld("weight", a.weight, a.in_dim, &a.ldw);
  c.ld("preact", a.preact, a.out_dim, &a.ldz);
  c.ld("dx", a.dx, a.in_dim, &a.lddx);
  c.ld("dweight", a.dweight, a.in_dim, &a.lddw);
  c.in("dy", a.dy, a.n, a.out_dim, a.lddy);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("weight", a.weight, a.out_dim, a.in_dim, a.ldw);
  c.in("preact", a.preact, a.n, a.out_dim, a.ldz);
  c.out("dx", a.dx, a.n, a.in_dim, a.lddx);
  c.out("dweight", a.dweight, a.out_dim, a.in_dim, a.lddw);
  c.out("dbias", a.dbias, 1, a.out_dim, a.out_dim);
  if ((st = c.overlaps())) return st;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  Backward b{};
  b.storage = a.storage, b.act = a.activation, b.parts = 1;
  b.n = a.n, b.in_dim = a.in_dim, b.out_dim = a.out_dim;
  b.dy = a.dy, b.x = a.x, b.w[0] = a.weight, b.pre[0] = a.preact;
  b.dx = a.dx, b.dw[0] = a.dweight, b.db[0] = a.dbias;
  b.lddy = a.lddy, b.ldx = a.ldx, b.ldw = a.ldw, b.ldpre = a.ldz, b.lddx = a.lddx, b.lddw = a.lddw;
  b.status = a.status, b.stream = static_cast<cudaStream_t>(a.stream);
  return run_backward(b);
}

extern "C" xvec_gpu_status xvec_gpu_gated_backward_device(
    const xvec_gpu_gated_backward_args* args) {
  xvec_gpu_status st = check_shape(args);
  if (st) return st;
  xvec_gpu_gated_backward_args a = *args;
  if (a.n && (!a.dh || !a.gate || !a.up)) return invalid("dh, gate and up are required");
  if (a.dx && (!a.gate_weight || !a.up_weight)) return invalid("dx needs both weights");
  if (a.n && (a.dgate_weight || a.dup_weight) && !a.x) return invalid("weight gradients need x");
  Check c(elem_bytes(a.storage));
  c.ld("dh", a.dh, a.out_dim, &a.lddh);
  c.ld("x", a.x, a.in_dim, &a.ldx);
  c.ld("the weights", a.gate_weight ? a.gate_weight : a.up_weight, a.in_dim, &a.ldw);
  c.ld("gate and up", a.gate, a.out_dim, &a.ldg);
  c.ld("dx", a.dx, a.in_dim, &a.lddx);
  c.ld("the weight gradients", a.dgate_weight ? a.dgate_weight : a.dup_weight, a.in_dim, &a.lddw);
  c.in("dh", a.dh, a.n, a.out_dim, a.lddh);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("gate_weight", a.gate_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("up_weight", a.up_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("gate", a.gate, a.n, a.out_dim, a.ldg);
  c.in("up", a.up, a.n, a.out_dim, a.ldg);
  c.out("dx", a.dx, a.n, a.in_dim, a.lddx);
  c.out("dgate_weight", a.dgate_weight, a.out_dim, a.in_dim, a.lddw);
  c.out("dup_weight", a.dup_weight, a.out_dim, a.in_dim, a.lddw);
  c.out("dgate_bias", a.dgate_bias, 1, a.out_dim, a.out_dim);
  c.out("dup_bias", a.dup_bias, 1, a.out_dim, a.out_dim);
  if ((st = c.overlaps())) return st;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  Backward b{};
  b.storage = a.storage, b.act = a.activation, b.parts = 2;
  b.n = a.n, b.in_dim = a.in_dim, b.out_dim = a.out_dim;
  b.dy = a.dh, b.x = a.x, b.w[0] = a.gate_weight, b.w[1] = a.up_weight;
  b.pre[0] = a.gate, b.pre[1] = a.up;
  b.dx = a.dx, b.dw[0] = a.dgate_weight, b.dw[1] = a.dup_weight;
  b.db[0] = a.dgate_bias, b.db[1] = a.dup_bias;
  b.lddy = a.lddh, b.ldx = a.ldx, b.ldw = a.ldw, b.ldpre = a.ldg, b.lddx = a.lddx, b.lddw = a.lddw;
  b.status = a.status, b.stream = static_cast<cudaStream_t>(a.stream);
  return run_backward(b);
}
