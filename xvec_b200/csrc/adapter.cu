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

// --- operands -----------------------------------------------------------------
// Eight values as operand elements at dst: 16-bit types as they are; float32
// as three bfloat16 parts x = h + m + l in planes `plane` elements apart, each
// the nearest to what is left (exact: 8 bits each and the parts' signs).
template <typename T>
__device__ __forceinline__ void store_operand(void* dst, int64_t plane, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    *static_cast<uint4*>(dst) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                           pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  } else {
    __align__(16) bf16 t[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = v[j];
      bf16 h = __float2bfloat16_rn(x);
      // Next to the largest float32 the nearest bfloat16 is an infinity.
      if (isinf(to_f(h)) && !isinf(x)) h = __float2bfloat16_rz(x);
      const bool finite = isfinite(x);
      x = finite ? x - to_f(h) : 0.f;
      const bf16 m = __float2bfloat16_rn(x);
      t[0][j] = h, t[1][j] = m, t[2][j] = __float2bfloat16_rn(x - to_f(m));
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(dst) + i * plane) =
          *reinterpret_cast<uint4*>(t[i]);
  }
}

// A [rows][cols] matrix to become an operand: contiguous rows of ld (a multiple
// of 8) elements, zeros behind the columns.
struct Pack {
  const void* src;
  void* dst;
  int64_t lds, rows, ld;
  int cols, vec;
};
struct Packs {
  Pack p[3];
  int n = 0;
};
// Packs up to three matrices (blockIdx.y) at once.  Bound by memory.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs packs) {
  pdl_begin();
  const Pack& p = packs.p[blockIdx.y];
  const T* src = static_cast<const T*>(p.src);
  const int64_t groups = p.ld / 8, total = groups * p.rows;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    // (64-bit divisions would cost more than the copy.)
    const int64_t r = total >> 32 ? i / groups : (uint32_t)i / (uint32_t)groups;
    const int c = (int)(i - r * groups) * 8;
    float v[8];
    load8(src + r * p.lds + c, p.cols - c, p.vec, v);
    store_operand<T>(static_cast<uint16_t*>(p.dst) + r * p.ld + c, p.rows * p.ld, v);
  }
}

size_t elem_bytes(int storage) { return storage == XVEC_STORAGE_FP32 ? 4 : 2; }
int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }
int planes_of(int storage) { return storage == XVEC_STORAGE_FP32 ? 3 : 1; }

unsigned grid_of(int64_t threads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 148 * 16));
}

// The operand for a [rows][cols] matrix: in place where the copies into shared
// memory can start on 16 bytes, else `room`, for run_packs to fill.
xvec_gpu_status operand(int storage, const void* p, int64_t rows, int64_t cols, int64_t ld,
                        Scratch* room, GemmOperand* out, Packs* packs, cudaStream_t s) {
  out->inner = cols, out->outer = rows;
  if (storage != XVEC_STORAGE_FP32 && aligned16(p, ld, 2)) {
    out->p = p, out->ld = ld, out->planes = 1;
    return XVEC_GPU_OK;
  }
  out->ld = round8(cols);
  out->plane = rows * out->ld;
  out->planes = planes_of(storage);
  if (xvec_gpu_status st = room->alloc((size_t)out->planes * out->plane * 2, s)) return st;
  out->p = room->ptr;
  packs->p[packs->n++] = {p, room->ptr, ld, rows, out->ld, (int)cols,
                          aligned16(p, ld, elem_bytes(storage)) ? 1 : 0};
  return XVEC_GPU_OK;
}
xvec_gpu_status run_packs(int storage, const Packs& packs, cudaStream_t s) {
  if (packs.n == 0) return XVEC_GPU_OK;
  int64_t most = 0;
  for (int i = 0; i < packs.n; ++i) most = std::max(most, packs.p[i].rows * packs.p[i].ld / 8);
  // 16-bit types: the bits pass through float and back, exactly but for the
  // payload of a NaN.
  auto* kern = storage == XVEC_STORAGE_FP32   ? pack_kernel<float>
               : storage == XVEC_STORAGE_FP16 ? pack_kernel<__half>
                                              : pack_kernel<bf16>;
  XVEC_CUDA(launch_pdl(kern, dim3(grid_of(most), packs.n), 256, 0, s, 1, packs));
  return XVEC_GPU_OK;
}

xvec_gpu_status gemm(int storage, GemmCall& c, cudaStream_t s) {
  c.bf16 = storage != XVEC_STORAGE_FP16;
  c.p.wait_ns = (uint64_t)wait_limit_ns();
  return storage == XVEC_STORAGE_FP32   ? gemm_fp32(c, s)
         : storage == XVEC_STORAGE_FP16 ? gemm_fp16(c, s)
                                        : gemm_bf16(c, s);
}

// --- pre-activation gradients and their column sums -----------------------
// dz = dy act'(z), or (GATED) dg = dh u act'(g) and du = dh act(g), as operands
// [2][planes][n][ld] (out may be NULL: column sums only); partial
// [2][chunks][m]: the column sums of each row chunk in float32, before any
// rounding.  A block owns 256 columns of a row chunk: 32 threads of 8 columns,
// 8 rows at a time.  Bound by memory.
template <typename T>
struct Eight {
  static constexpr int N = sizeof(T) / 2;  // 16-byte parts
  uint4 v[N];
  __device__ __forceinline__ void load(const T* p, int count, bool vec) {
    if (vec && count >= 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
      T* t = reinterpret_cast<T*>(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = j < count ? p[j] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    return to_f(reinterpret_cast<const T*>(v)[j]);
  }
};

// kRows rows of a thread are requested before the first is used and held as
// they came.  (Held as floats they took 122 registers, a quarter of the warps.)
template <typename T, bool GATED>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
    slope_kernel(const T* dy, int64_t lddy, const T* z, const T* u, int64_t ldz, int64_t n, int m,
                 int act, int vec, int64_t rows_per_chunk, uint16_t* out, int64_t ld,
                 float* partial) {
  pdl_begin();
  constexpr int kOuts = GATED ? 2 : 1;
  constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
  constexpr int kRows = 2;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 256 + tx * 8;
  const int64_t r0 = blockIdx.y * rows_per_chunk;
  const int64_t r1 = min(n, r0 + rows_per_chunk);
  const bool act_needed = GATED || act != XVEC_ACT_NONE;
  float sum[kOuts][8] = {};
  if (c < m) {
    for (int64_t r = r0 + ty; r < r1; r += 8 * kRows) {
      Eight<T> dr[kRows], zr[kRows], ur[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t q = r + 8 * i < r1 ? r + 8 * i : r;
        dr[i].load(dy + q * lddy + c, m - c, vec & 1);
        if (act_needed) zr[i].load(z + q * ldz + c, m - c, vec & 2);
        if (GATED) ur[i].load(u + q * ldz + c, m - c, vec & 4);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (r + 8 * i >= r1) break;
        float d[kOuts][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d[0][j] = dr[i][j];
          if (act_needed) {
            float slope;
            const float a = activate_slope<T>(act, zr[i][j], &slope);
            if constexpr (GATED) {
              d[1][j] = d[0][j] * a;
              d[0][j] *= ur[i][j];
            }
            d[0][j] *= slope;
          }
        }
#pragma unroll
        for (int o = 0; o < kOuts; ++o) {
          if (out)
            store_operand<T>(out + (o * kPlanes * n + r + 8 * i) * ld + c, n * ld, d[o]);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[o][j] += d[o][j];
        }
      }
    }
  }
  if (partial) {
    __shared__ float part[8][256];
#pragma unroll
    for (int o = 0; o < kOuts; ++o) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) part[ty][tx * 8 + j] = sum[o][j];
      __syncthreads();
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
      const int col = blockIdx.x * 256 + threadIdx.x;
      if (col < m) partial[((int64_t)o * gridDim.y + blockIdx.y) * m + col] = s;
    }
  }
}

// out[c] = the sum over the chunks in a fixed order: 32 interleaved runs, then
// those.
constexpr int kSumThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kSumThreads)
    column_sum_kernel(const float* partial, int chunks, int m, T* out0, T* out1) {
  pdl_begin();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  T* out = blockIdx.y ? out1 : out0;
  if (!out) return;
  const float* p = partial + (int64_t)blockIdx.y * chunks * m + c;
  float s = 0.f;
  if (c < m)
    for (int i = ty; i < chunks; i += 32) s += p[(int64_t)i * m];
  __shared__ float part[32][33];
  part[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < m) {
    for (int i = 1; i < 32; ++i) s += part[i][tx];
    out[c] = from_f<T>(s);
  }
}

// The pre-activation gradients of one backward call.
struct Slopes {
  const void *dy, *z, *u;  // u: gated only
  int64_t lddy, ldz, n;
  int m, act;
  void* out;  // NULL: not wanted
  int64_t ld;
  void* db[2];
};

template <typename T>
xvec_gpu_status slopes_t(const Slopes& a, cudaStream_t s) {
  const int cols = (a.m + 255) / 256;
  const bool sums = a.db[0] || a.db[1];
  // About eight blocks per SM, of at least 16 rows.
  const int64_t chunks =
      std::max<int64_t>(1, std::min<int64_t>((a.n + 15) / 16, std::max(1, 148 * 8 / cols)));
  const int64_t per = ((a.n + chunks - 1) / chunks + 15) / 16 * 16;
  const int used = (int)((a.n + per - 1) / per);
  Scratch partial;
  if (sums)
    if (xvec_gpu_status st = partial.alloc((size_t)2 * used * a.m * 4, s)) return st;
  const int vec = (aligned16(a.dy, a.lddy, sizeof(T)) ? 1 : 0) |
                  (aligned16(a.z, a.ldz, sizeof(T)) ? 2 : 0) |
                  (aligned16(a.u, a.ldz, sizeof(T)) ? 4 : 0);
  auto* kern = a.u ? slope_kernel<T, true> : slope_kernel<T, false>;
  XVEC_CUDA(launch_pdl(kern, dim3(cols, used), 256, 0, s, 1, static_cast<const T*>(a.dy), a.lddy,
                       static_cast<const T*>(a.z), static_cast<const T*>(a.u), a.ldz, a.n, a.m,
                       a.act, vec, per, static_cast<uint16_t*>(a.out), a.ld, partial.as<float>()));
  if (sums)
    XVEC_CUDA(launch_pdl(column_sum_kernel<T>, dim3((a.m + 31) / 32, 2), kSumThreads, 0, s, 1,
                         partial.as<float>(), used, a.m, static_cast<T*>(a.db[0]),
                         static_cast<T*>(a.db[1])));
  return XVEC_GPU_OK;
}

xvec_gpu_status slopes(int storage, const Slopes& a, cudaStream_t s) {
  return storage == XVEC_STORAGE_FP32   ? slopes_t<float>(a, s)
         : storage == XVEC_STORAGE_FP16 ? slopes_t<__half>(a, s)
                                        : slopes_t<bf16>(a, s);
}

// --- argument checks --------------------------------------------------------
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
  cudaStream_t s = static_cast<cudaStream_t>(a.stream);
  if (a.n <= kFewRows) {
    FewRows f{};
    f.n = (int)a.n, f.in_dim = a.in_dim, f.out_dim = a.out_dim, f.act = a.activation;
    f.x = a.x, f.w[0] = a.weight, f.bias[0] = a.bias, f.residual = a.residual;
    f.out = a.y, f.save[0] = a.preact;
    f.ldx = a.ldx, f.ldw = a.ldw, f.ldr = a.ldr, f.ldo = a.ldy, f.lds = a.ldz;
    return few_rows(a.storage, f, s);
  }
  GemmCall g;
  g.mode = kLinear;
  g.depth = a.in_dim;
  Scratch room[2];
  Packs packs;
  if ((st = operand(a.storage, a.x, a.n, a.in_dim, a.ldx, &room[0], &g.a, &packs, s)) ||
      (st = operand(a.storage, a.weight, a.out_dim, a.in_dim, a.ldw, &room[1], &g.b[0], &packs,
                    s)) ||
      (st = run_packs(a.storage, packs, s)))
    return st;
  GemmParams& p = g.p;
  p.rows = a.n, p.cols = a.out_dim, p.segs = p.batches = 1;
  p.bias[0] = a.bias;
  p.residual = a.residual, p.ldr = a.ldr;
  p.out[0] = a.y, p.ldo = a.ldy;
  p.save[0] = a.preact, p.lds = a.ldz;
  p.act = a.activation;
  p.status = a.status;
  const size_t size = elem_bytes(a.storage);
  p.vec = aligned16(a.y, a.ldy, size) && aligned16(a.residual, a.ldr, size) &&
          aligned16(a.preact, a.ldz, size);
  return gemm(a.storage, g, s);
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
  cudaStream_t s = static_cast<cudaStream_t>(a.stream);
  if (a.n <= kFewRows) {
    FewRows f{};
    f.n = (int)a.n, f.in_dim = a.in_dim, f.out_dim = a.out_dim, f.act = a.activation;
    f.x = a.x, f.w[0] = a.gate_weight, f.w[1] = a.up_weight;
    f.bias[0] = a.gate_bias, f.bias[1] = a.up_bias;
    f.out = a.h, f.save[0] = a.gate, f.save[1] = a.up;
    f.ldx = a.ldx, f.ldw = a.ldw, f.ldo = a.ldh, f.lds = a.ldg;
    return few_rows(a.storage, f, s);
  }
  GemmCall g;
  g.mode = kGated;
  g.depth = a.in_dim;
  Scratch room[3];
  Packs packs;
  if ((st = operand(a.storage, a.x, a.n, a.in_dim, a.ldx, &room[0], &g.a, &packs, s)) ||
      (st = operand(a.storage, a.gate_weight, a.out_dim, a.in_dim, a.ldw, &room[1], &g.b[0],
                    &packs, s)) ||
      (st = operand(a.storage, a.up_weight, a.out_dim, a.in_dim, a.ldw, &room[2], &g.b[1], &packs,
                    s)) ||
      (st = run_packs(a.storage, packs, s)))
    return st;
  GemmParams& p = g.p;
  p.rows = a.n, p.cols = a.out_dim, p.segs = p.batches = 1;
  p.bias[0] = a.gate_bias, p.bias[1] = a.up_bias;
  p.out[0] = a.h, p.ldo = a.ldh;
  p.save[0] = a.gate, p.save[1] = a.up, p.lds = a.ldg;
  p.act = a.activation;
  p.status = a.status;
  const size_t size = elem_bytes(a.storage);
  p.vec = aligned16(a.h, a.ldh, size) && aligned16(a.gate, a.ldg, size) &&
          aligned16(a.up, a.ldg, size);
  return gemm(a.storage, g, s);
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
  if (b.n == 0) {
    for (int i = 0; i < b.parts; ++i) {
      if (b.dw[i])
        XVEC_CUDA(cudaMemset2DAsync(b.dw[i], b.lddw * size, 0, b.in_dim * size, b.out_dim, s));
      if (b.db[i]) XVEC_CUDA(cudaMemsetAsync(b.db[i], 0, b.out_dim * size, s));
    }
    return XVEC_GPU_OK;
  }
  const bool products = b.dx || b.dw[0] || b.dw[1], sums = b.db[0] || b.db[1];
  if (!products && !sums) return XVEC_GPU_OK;
  // The pre-activation gradients as one operand of `parts` matrices.  dy itself
  // where no activation changes it and it can be read in place.
  Scratch dz;
  GemmOperand grad;
  grad.inner = b.out_dim, grad.outer = b.n;
  const bool direct = b.parts == 1 && b.act == XVEC_ACT_NONE && size == 2 &&
                      aligned16(b.dy, b.lddy, size);
  if (direct) {
    grad.p = b.dy, grad.ld = b.lddy;
  } else {
    grad.ld = round8(b.out_dim);
    grad.plane = b.n * grad.ld;
    grad.planes = planes_of(b.storage) * b.parts;
    if (products) {
      if ((st = dz.alloc((size_t)grad.planes * grad.plane * 2, s))) return st;
      grad.p = dz.ptr;
    }
  }
  if (!direct || sums) {
    Slopes a{};
    a.dy = b.dy, a.z = b.pre[0], a.u = b.pre[1];
    a.lddy = b.lddy, a.ldz = b.ldpre, a.n = b.n, a.m = b.out_dim, a.act = b.act;
    a.out = dz.ptr, a.ld = grad.ld;
    a.db[0] = b.db[0], a.db[1] = b.db[1];
    if ((st = slopes(b.storage, a, s))) return st;
  }
  Scratch room[3];
  GemmOperand w[2], x;
  Packs packs;
  if (b.dx)
    for (int i = 0; i < b.parts; ++i)
      if ((st = operand(b.storage, b.w[i], b.out_dim, b.in_dim, b.ldw, &room[i], &w[i], &packs, s)))
        return st;
  if (b.dw[0] || b.dw[1])
    if ((st = operand(b.storage, b.x, b.n, b.in_dim, b.ldx, &room[2], &x, &packs, s))) return st;
  if ((st = run_packs(b.storage, packs, s))) return st;
  if (b.dx) {
    GemmCall g;
    g.mode = kDx;
    g.depth = b.out_dim;
    g.a = grad;
    for (int i = 0; i < b.parts; ++i) g.b[i] = w[i];
    g.p.rows = b.n, g.p.cols = b.in_dim, g.p.segs = b.parts, g.p.batches = 1;
    g.p.out[0] = b.dx, g.p.ldo = b.lddx;
    g.p.vec = aligned16(b.dx, b.lddx, size);
    g.p.status = b.status;
    if ((st = gemm(b.storage, g, s))) return st;
  }
  if (b.dw[0] || b.dw[1]) {
    GemmCall g;
    g.mode = kDw;
    g.depth = b.n;
    g.a = grad;
    g.b[0] = x;
    g.p.rows = b.out_dim, g.p.cols = b.in_dim, g.p.segs = 1;
    g.p.vec = 1;
    // Only the second weight's gradient: start at its matrix.
    const int first = b.dw[0] ? 0 : 1;
    if (first) {
      g.a.p = static_cast<const uint16_t*>(grad.p) + planes_of(b.storage) * grad.plane;
      g.a.planes = planes_of(b.storage);
    }
    for (int i = first; i < b.parts && b.dw[i]; ++i) {
      g.p.out[g.p.batches++] = b.dw[i];
      g.p.vec &= aligned16(b.dw[i], b.lddw, size);
    }
    g.p.ldo = b.lddw;
    g.p.status = b.status;
    if ((st = gemm(b.storage, g, s))) return st;
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
