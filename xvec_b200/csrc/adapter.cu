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
#include <cfloat>
#include <climits>
#include <mutex>

#include "adapter.cuh"

namespace xvec {
namespace adapter {
namespace {

constexpr int64_t kMaxDim = 1 << 20;
constexpr int kMaxDevices = 64;
// What of freed scratch stays with the library for the next calls.  (Giving it back and
// taking it again costs 6 ms a GiB: a float32 weight gradient of 400,000 rows, 6.9 GiB, whose
// caller waits after every call took 46 ms instead of 6.8 with 4 GiB kept.)
constexpr uint64_t kScratchKept = 16ull << 30;

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
template <typename T, bool VEC>
__device__ __forceinline__ void pack_rows(const Pack& p, int64_t thread, int64_t threads) {
  const T* src = static_cast<const T*>(p.src);
  const int64_t groups = p.ld / 8, total = groups * p.rows;
  constexpr int kAhead = 2;  // groups requested before the first is stored
  for (int64_t i0 = thread; i0 < total; i0 += kAhead * threads) {
    Eight<T, VEC> e[kAhead];
    int64_t r[kAhead];
    int c[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t i = i0 + a * threads < total ? i0 + a * threads : i0;
      // (64-bit divisions would cost more than the copy.)
      r[a] = total >> 32 ? i / groups : (uint32_t)i / (uint32_t)groups;
      c[a] = (int)(i - r[a] * groups) * 8;
      e[a].load(src + r[a] * p.lds + c[a], p.cols - c[a]);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i0 + a * threads >= total) break;
      e[a].settle();
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c[a] + j < p.cols ? e[a][j] : 0.f;
      store_operand<T>(static_cast<uint16_t*>(p.dst) + r[a] * p.ld + c[a], p.rows * p.ld, v);
    }
  }
}
template <typename T>
__device__ __forceinline__ void pack(const Pack& p, int64_t thread, int64_t threads) {
  if (p.vec) pack_rows<T, true>(p, thread, threads);
  else pack_rows<T, false>(p, thread, threads);
}
// Packs up to three matrices (blockIdx.y) at once.  Bound by memory.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs packs) {
  pdl_begin();
  pack<T>(packs.p[blockIdx.y], (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

size_t elem_bytes(int storage) { return storage == XVEC_STORAGE_FP32 ? 4 : 2; }
int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }
int planes_of(int storage) { return storage == XVEC_STORAGE_FP32 ? 3 : 1; }

unsigned grid_of(int64_t threads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 148 * 16));
}

// One call's scratch: a single stream-ordered allocation, handed out in parts.
struct Arena {
  Scratch room;
  size_t used = 0;
  size_t add(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
  xvec_gpu_status alloc(const DeviceGuard& guard, cudaStream_t s) {
    return used ? room.alloc(used, s, guard.pool) : XVEC_GPU_OK;
  }
  void* at(size_t offset) const { return room.as<char>() + offset; }
};

// The operand for a [rows][cols] matrix: in place where the copies into shared
// memory can start on 16 bytes, else a place in the arena for the packing.
// (16-bit types: packed bits pass through float and back, exactly but for the
// payload of a NaN.)
struct Operand {
  GemmOperand g;
  bool packed = false;
  size_t at = 0;
  Pack pack{};
};
Operand plan_operand(int storage, const void* p, int64_t rows, int64_t cols, int64_t ld,
                     Arena* arena) {
  Operand o;
  o.g.p = p, o.g.inner = cols, o.g.outer = rows, o.g.ld = ld;
  if (storage != XVEC_STORAGE_FP32 && aligned16(p, ld, 2)) return o;
  o.packed = true;
  o.g.ld = round8(cols);
  o.g.plane = rows * o.g.ld;
  o.g.planes = planes_of(storage);
  o.at = arena->add((size_t)o.g.planes * o.g.plane * 2);
  o.pack = {p, nullptr, ld, rows, o.g.ld, (int)cols, aligned16(p, ld, elem_bytes(storage)) ? 1 : 0};
  return o;
}
// Once the arena is there.
void place(Operand* o, const Arena& arena, Packs* packs) {
  if (!o->packed) return;
  o->g.p = o->pack.dst = arena.at(o->at);
  packs->p[packs->n++] = o->pack;
}
xvec_gpu_status run_packs(int storage, const Packs& packs, cudaStream_t s) {
  if (packs.n == 0) return XVEC_GPU_OK;
  int64_t most = 0;
  for (int i = 0; i < packs.n; ++i) most = std::max(most, packs.p[i].rows * packs.p[i].ld / 8);
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

// A forward product: plan, scratch, packing, launch.
xvec_gpu_status forward(int storage, GemmCall& g, Operand* a, Operand* b0, Operand* b1, Arena& arena,
                        const DeviceGuard& guard, cudaStream_t s) {
  xvec_gpu_status st = plan_gemm(storage, &g);
  if (st) return st;
  const size_t partial = arena.add(g.partial_bytes), runs = arena.add(g.run_bytes);
  if ((st = arena.alloc(guard, s))) return st;
  Packs packs;
  place(a, arena, &packs);
  place(b0, arena, &packs);
  if (b1) place(b1, arena, &packs);
  if ((st = run_packs(storage, packs, s))) return st;
  g.a = a->g, g.b[0] = b0->g;
  if (b1) g.b[1] = b1->g;
  if (g.partial_bytes) g.p.partial = static_cast<float*>(arena.at(partial));
  if (g.run_bytes) g.p.runs = static_cast<float*>(arena.at(runs));
  return gemm(storage, g, s);
}

// --- pre-activation gradients and their column sums -----------------------
// 16-bit storage rounds them to its type, since they are operands of two products: dx and
// the weight gradients are then off by sqrt(2) of one rounding (2.9e-4 of the 2-norm for
// binary16, where the results' own rounding leaves 2.1e-4).  A second 16-bit part would take
// that back and double the products, 190 of the 270 us of 8192 x 1024 -> 4096 gated.  The
// column sums add the gradients before any rounding.
// One backward call's: dz = dy act'(z), or dg = dh u act'(g) and du = dh act(g), as
// operands [2][planes][n][ld] (out may be NULL: column sums only); partial
// [2][chunks][m]: the column sums of each row chunk in float32, before any
// rounding; and the call's packings.
struct Slopes {
  const void *dy, *z, *u;  // u: gated only
  int64_t lddy, ldz, n;
  int m, act;
  int cols, chunks;  // blocks: of 256 columns, of rows_per_chunk rows
  int64_t rows_per_chunk;
  uint16_t* out;
  int64_t ld;
  float* partial;
  float* peaks;  // [cols chunks] each block's largest finite |gradient| (binary16 operands)
  float* scale;  // what the operands' products are multiplied by (AGAIN)
  Packs packs;
  unsigned pack_blocks;  // for each packing
};

// --- the scale of binary16 operands
// The least largest value that needs no scaling: binary16 holds what is 2^-8 of it in full.
constexpr float kLeastPeak = 0.015625f;
// The largest v of the block's 256 threads, on every thread.
__device__ __forceinline__ float block_max(float v) {
  __shared__ float part[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) v = fmaxf(v, part[i]);
  return v;
}
// The power of two that the operands are multiplied by.
__device__ __forceinline__ float operand_scale(const float* peaks, int num) {
  float peak = 0.f;
  for (int i = threadIdx.x; i < num; i += 256) peak = fmaxf(peak, peaks[i]);
  peak = block_max(peak);
  if (peak == 0.f || (peak >= kLeastPeak && peak <= 65504.f)) return 1.f;
  return ldexpf(1.f, min(14 - ilogbf(peak), 126));
}

// Blocks [0, cols chunks) are the gradients', the others the packings'.  A block
// owns 256 columns of a row chunk: 32 threads of 8 columns, 8 rows at a time; bound
// by memory (8192 x 4096 fp16 gated: 53 us, 335 MB).
// kRows rows of a thread are requested before the first is used and held as
// they came.  (Held as floats they took 122 registers, a quarter of the warps.)
// VEC: all of dy, z and u allow 16-byte accesses.
// AGAIN: after a first pass, binary16 operands only.  A gradient of two or three stored
// values easily leaves binary16's range where its products do not.  If the largest is
// outside kLeastPeak..65504, the operands are written once more, times the power of two
// that brings it to 2^14..2^15; values below 2^-40 of it are lost.  Else nothing but
// *scale = 1 is left to do (4 us; the maxima cost the first pass 4 us of 54).
template <typename T, bool GATED, bool VEC, bool AGAIN>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : VEC ? 4 : 3)
    slope_kernel(const __grid_constant__ Slopes p) {
  pdl_begin();
  float up = 1.f;
  if constexpr (AGAIN) {
    up = operand_scale(p.peaks, p.cols * p.chunks);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.scale = 1.f / up;  // (a power of two)
    if (up == 1.f) return;
  }
  const unsigned slope_blocks = (unsigned)p.cols * p.chunks;
  if (!AGAIN && blockIdx.x >= slope_blocks) {
    const unsigned b = blockIdx.x - slope_blocks, which = b / p.pack_blocks;
    pack<T>(p.packs.p[which], (int64_t)(b - which * p.pack_blocks) * 256 + threadIdx.x,
            (int64_t)p.pack_blocks * 256);
    return;
  }
  const unsigned chunk = blockIdx.x / p.cols, col_block = blockIdx.x - chunk * p.cols;
  const T* dy = static_cast<const T*>(p.dy);
  const T* z = static_cast<const T*>(p.z);
  const T* u = static_cast<const T*>(p.u);
  const int64_t lddy = p.lddy, ldz = p.ldz, n = p.n, ld = p.ld;
  const int m = p.m, act = p.act;
  uint16_t* out = p.out;
  constexpr int kOuts = GATED ? 2 : 1;
  constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
  constexpr int kRows = 2;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = col_block * 256 + tx * 8;
  const int64_t r0 = chunk * p.rows_per_chunk;
  const int64_t r1 = min(n, r0 + p.rows_per_chunk);
  const bool act_needed = GATED || act != XVEC_ACT_NONE;
  constexpr bool kPeak = std::is_same<T, __half>::value && !AGAIN;
  float sum[kOuts][8] = {}, peak = 0.f;
  if (c < m) {
    for (int64_t r = r0 + ty; r < r1; r += 8 * kRows) {
      Eight<T, VEC> dr[kRows], zr[kRows], ur[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t q = r + 8 * i < r1 ? r + 8 * i : r;
        dr[i].load(dy + q * lddy + c, m - c);
        if (act_needed) zr[i].load(z + q * ldz + c, m - c);
        if (GATED) ur[i].load(u + q * ldz + c, m - c);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (r + 8 * i >= r1) break;
        dr[i].settle();
        if (act_needed) zr[i].settle();
        if (GATED) ur[i].settle();
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
          if constexpr (AGAIN) {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[o][j] *= up;
          }
          if (out)
            store_operand<T>(out + (o * kPlanes * n + r + 8 * i) * ld + c, n * ld, d[o]);
          if constexpr (kPeak) {
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(d[o][j]));
            if (most > FLT_MAX || m - c < 8) {  // only what is finite and exists
              most = 0.f;
              for (int j = 0; j < 8; ++j)
                if (fabsf(d[o][j]) <= FLT_MAX && c + j < m) most = fmaxf(most, fabsf(d[o][j]));
            }
            peak = fmaxf(peak, most);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[o][j] += d[o][j];
        }
      }
    }
  }
  if constexpr (kPeak) {
    if (p.peaks) {
      peak = block_max(peak);
      if (threadIdx.x == 0) p.peaks[blockIdx.x] = peak;
    }
  }
  if (!AGAIN && p.partial) {
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
      const int col = col_block * 256 + threadIdx.x;
      if (col < m) p.partial[((int64_t)o * p.chunks + chunk) * m + col] = s;
    }
  }
}

// The row chunks' column sums alone, where dy is its own gradient and read in place:
// as above, with eight rows of a thread on their way (two: 14 us for 16384 x 1024
// bfloat16; eight: 9).
template <typename T>
__global__ void __launch_bounds__(256, 4) chunk_sum_kernel(const __grid_constant__ Slopes p) {
  pdl_begin();
  constexpr int kRows = 8;
  const unsigned chunk = blockIdx.x / p.cols, col_block = blockIdx.x - chunk * p.cols;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = col_block * 256 + tx * 8;
  const int64_t r0 = chunk * p.rows_per_chunk, r1 = min(p.n, r0 + p.rows_per_chunk);
  const T* dy = static_cast<const T*>(p.dy);
  float sum[8] = {};
  if (c < p.m) {
    for (int64_t r = r0 + ty; r < r1; r += 8 * kRows) {
      Eight<T, true> d[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t q = r + 8 * i;
        d[i].load(dy + (q < r1 ? q : r) * p.lddy + c, p.m - c);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (r + 8 * i < r1)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += d[i][j];
    }
  }
  __shared__ float part[8][256];
#pragma unroll
  for (int j = 0; j < 8; ++j) part[ty][tx * 8 + j] = sum[j];
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
  const int col = col_block * 256 + threadIdx.x;
  if (col < p.m) p.partial[(int64_t)chunk * p.m + col] = s;
}

// The column sums alone, where no product follows that could take them along.
template <typename T>
__global__ void __launch_bounds__(128)
    column_sum_kernel(const float* sums, int chunks, int m, void* out0, void* out1) {
  pdl_begin();
  column_sums<T>(sums, chunks, m, out0, out1, blockIdx.x * 4 + (threadIdx.x >> 5), gridDim.x * 4,
                 threadIdx.x & 31);
}

// Row chunks of the gradient pass: about eight blocks per SM, of at least 16 rows and
// at most 2048 (a thread then adds 256 values in a row).
void plan_slopes(Slopes* a) {
  a->cols = (a->m + 255) / 256;
  const int64_t most =
      std::min<int64_t>((a->n + 15) / 16,
                        std::max<int64_t>((a->n + 2047) / 2048, 148 * 8 / a->cols));
  a->rows_per_chunk = ((a->n + most - 1) / most + 15) / 16 * 16;  // (n >= 1)
  a->chunks = (int)((a->n + a->rows_per_chunk - 1) / a->rows_per_chunk);
}

template <typename T>
xvec_gpu_status slopes_t(Slopes& a, cudaStream_t s) {
  const bool vec = aligned16(a.dy, a.lddy, sizeof(T)) &&
                   (aligned16(a.z, a.ldz, sizeof(T)) || (!a.u && a.act == XVEC_ACT_NONE)) &&
                   (!a.u || aligned16(a.u, a.ldz, sizeof(T)));
  int64_t most = 0;
  for (int i = 0; i < a.packs.n; ++i)
    most = std::max(most, a.packs.p[i].rows * a.packs.p[i].ld / 8);
  a.pack_blocks = grid_of(most);
  auto* kern = a.u ? (vec ? slope_kernel<T, true, true, false> : slope_kernel<T, true, false, false>)
                   : (vec ? slope_kernel<T, false, true, false> : slope_kernel<T, false, false, false>);
  const unsigned blocks = (unsigned)a.cols * a.chunks;
  XVEC_CUDA(launch_pdl(kern, dim3(blocks + a.pack_blocks * a.packs.n), 256, 0, s, 1, a));
  if constexpr (std::is_same<T, __half>::value) {
    if (a.peaks) {
      auto* again = a.u ? (vec ? slope_kernel<T, true, true, true> : slope_kernel<T, true, false, true>)
                        : (vec ? slope_kernel<T, false, true, true> : slope_kernel<T, false, false, true>);
      XVEC_CUDA(launch_pdl(again, dim3(blocks), 256, 0, s, 1, a));
    }
  }
  return XVEC_GPU_OK;
}

xvec_gpu_status slopes(int storage, Slopes& a, cudaStream_t s) {
  return storage == XVEC_STORAGE_FP32   ? slopes_t<float>(a, s)
         : storage == XVEC_STORAGE_FP16 ? slopes_t<__half>(a, s)
                                        : slopes_t<bf16>(a, s);
}

// dy 16-bit and aligned.
xvec_gpu_status chunk_sums(int storage, const Slopes& a, cudaStream_t s) {
  auto* kern = storage == XVEC_STORAGE_FP16 ? chunk_sum_kernel<__half> : chunk_sum_kernel<bf16>;
  XVEC_CUDA(launch_pdl(kern, dim3((unsigned)a.cols * a.chunks), 256, 0, s, 1, a));
  return XVEC_GPU_OK;
}

xvec_gpu_status sum_columns(int storage, const GemmParams& p, cudaStream_t s) {
  auto* kern = storage == XVEC_STORAGE_FP32   ? column_sum_kernel<float>
               : storage == XVEC_STORAGE_FP16 ? column_sum_kernel<__half>
                                              : column_sum_kernel<bf16>;
  XVEC_CUDA(launch_pdl(kern, dim3((unsigned)std::min((p.sum_cols + 15) / 16, 1184)), 128, 0, s, 1,
                       p.sums, p.sum_chunks, p.sum_cols, p.sum_out[0], p.sum_out[1]));
  return XVEC_GPU_OK;
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

  // (The leading dimension of a single row means nothing.)
  void ld(const char* name, const void* p, int64_t rows, int64_t cols, int64_t* ld) {
    if (st || !p) return;
    if (*ld == 0 || rows <= 1) *ld = cols;
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
  void status(const int32_t* p) { out("status", p, 1, 4 / size, 4 / size); }
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
  if ((uintptr_t)a->status % 4) return invalid("status is not aligned");
  return XVEC_GPU_OK;
}

}  // namespace

// Tile shape and depth splits by a cost estimate in SM clocks: a wave's blocks
// and epilogue (which overlap in time but share shared memory and power: their
// times were seen to add up), a start, and for splits the traffic of their partial
// sums and a second launch.  A block takes 512 clocks for a pair's 256 columns (the
// matrix rate), 448 for 192, 384 for 128 (shared memory's rate), 590 for a single
// CTA's 128 x 128.  An epilogue column takes about 10 clocks for each matrix that
// it reads or writes and for an activation, up to 25 where rows do not allow
// 16-byte accesses.  192 columns exist for one product along depth (kLinear), where they can
// fill the last wave better: 10000 x 960 -> 960 fp32 is 200 tiles of three waves
// instead of 160 larger ones of three.
xvec_gpu_status plan_gemm(int storage, GemmCall* c) {
  const double products = storage == XVEC_STORAGE_FP32 ? 6 : 1;
  const double block[kShapes] = {512 * products, 448 * products, 384 * products, 590 * products};
  const double start[kShapes] = {7500, 7500, 7500, 3000};
  XVEC_CUDA(cudaGetDevice(&c->device));
  if (xvec_gpu_status st = count_sms(c->device, &c->sms)) return st;
  GemmParams& p = c->p;
  p.blocks = (int)((c->depth + 63) / 64);
  p.ldp = (p.cols + 63) / 64 * 64;  // whole steps of the epilogue
  const int all = p.blocks * p.segs;
  const int half = c->mode == kGated ? 2 : 1;  // accumulator columns per output column
  const int matrices = 1 + (p.save[0] != nullptr) + (p.save[1] != nullptr) +
                       (p.residual != nullptr) + (p.act != XVEC_ACT_NONE);
  double best = 0;
  p.splits = 0;
  for (int k = 0; k < kShapes; ++k) {
    if (k == 1 && c->mode != kLinear) continue;
    const int rows = kTileShapes[k].rows, cols = kTileShapes[k].cols / half;
    const int workers = kTileShapes[k].pair ? c->sms / 2 : c->sms;
    const int64_t tm = (p.rows + rows - 1) / rows, tn = (p.cols + cols - 1) / cols;
    for (int splits = 1; splits <= 32; ++splits) {
      const int per = (all + splits - 1) / splits;
      if (splits > 1 && (per * products < 4 || (int64_t)per * (splits - 1) >= all)) continue;
      const double waves = (double)((tm * tn * p.batches * splits + workers - 1) / workers);
      const double epilogue =
          cols * (splits > 1 ? 25.0 * half : matrices * (p.vec == 16 ? 10.0 : p.vec >= 4 ? 14.0 : 25.0));
      double cost = waves * (per * block[k] + epilogue) + start[k];
      if (splits > 1)
        cost += 6000 + (double)splits * p.rows * p.ldp * p.batches * half * 8 / 2000;
      if (p.splits == 0 || cost < best) {
        best = cost;
        c->shape = k;
        p.tiles_m = (int)tm, p.tiles_n = (int)tn, p.splits = splits, p.blocks_per_split = per;
      }
    }
  }
  c->partial_bytes =
      p.splits > 1 ? (size_t)p.splits * p.batches * half * p.rows * p.ldp * 4 : 0;
  // 128 rows of accumulator columns for each CTA.
  c->run_bytes = storage == XVEC_STORAGE_FP32 && p.blocks_per_split > run_blocks(true)
                     ? (size_t)c->sms * kTileShapes[c->shape].cols * 128 * 4
                     : 0;
  return XVEC_GPU_OK;
}

xvec_gpu_status count_sms(int device, int* sms) {
  static std::atomic<int> known[kMaxDevices];
  if (device < kMaxDevices && (*sms = known[device].load(std::memory_order_relaxed)))
    return XVEC_GPU_OK;
  XVEC_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
  if (device < kMaxDevices) known[device].store(*sms, std::memory_order_relaxed);
  return XVEC_GPU_OK;
}

DeviceGuard::~DeviceGuard() {
  if (relaxed) cudaThreadExchangeStreamCaptureMode(&mode);
  if (before >= 0) cudaSetDevice(before);
}

xvec_gpu_status DeviceGuard::set(int device) {
  static std::atomic<bool> ready[kMaxDevices];
  static cudaMemPool_t pools[kMaxDevices];
  static std::mutex first;
  const bool known =
      device >= 0 && device < kMaxDevices && ready[device].load(std::memory_order_acquire);
  int count = 0;
  if (!known && (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count)) {
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
  XVEC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  relaxed = true;
  if (known) {
    pool = pools[device];
    return XVEC_GPU_OK;
  }
  int major = 0, minor = 0;
  XVEC_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
  XVEC_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
  if (major != 10 || minor != 0) {
    set_error("device %d is not an sm_100 (B200) device", device);
    return XVEC_GPU_UNSUPPORTED;
  }
  if (device >= kMaxDevices) return XVEC_GPU_OK;  // (the default pool)
  // A pool of the library's own, so that the default pool stays as the caller set it up.
  std::lock_guard<std::mutex> lock(first);
  if (!ready[device].load(std::memory_order_relaxed)) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = device;
    cudaMemPool_t made;
    XVEC_CUDA(cudaMemPoolCreate(&made, &props));
    uint64_t kept = kScratchKept;
    XVEC_CUDA(cudaMemPoolSetAttribute(made, cudaMemPoolAttrReleaseThreshold, &kept));
    pools[device] = made;
    ready[device].store(true, std::memory_order_release);
  }
  pool = pools[device];
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
  c.ld("x", a.x, a.n, a.in_dim, &a.ldx);
  c.ld("weight", a.weight, a.out_dim, a.in_dim, &a.ldw);
  c.ld("residual", a.residual, a.n, a.out_dim, &a.ldr);
  c.ld("y", a.y, a.n, a.out_dim, &a.ldy);
  c.ld("preact", a.preact, a.n, a.out_dim, &a.ldz);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("weight", a.weight, a.out_dim, a.in_dim, a.ldw);
  c.in("bias", a.bias, 1, a.out_dim, a.out_dim);
  const char *y = "y", *residual = "residual";
  c.in(residual, a.residual, a.n, a.out_dim, a.ldr);
  c.out(y, a.y, a.n, a.out_dim, a.ldy);
  c.out("preact", a.preact, a.n, a.out_dim, a.ldz);
  c.status(a.status);
  if ((st = c.overlaps(y, residual))) return st;
  if (a.n == 0) return XVEC_GPU_OK;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  cudaStream_t s = static_cast<cudaStream_t>(a.stream);
  if (use_few_rows(a.storage, a.n, a.in_dim, a.out_dim, 1)) {
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
  Arena arena;
  Operand x = plan_operand(a.storage, a.x, a.n, a.in_dim, a.ldx, &arena);
  Operand w = plan_operand(a.storage, a.weight, a.out_dim, a.in_dim, a.ldw, &arena);
  GemmParams& p = g.p;
  p.rows = a.n, p.cols = a.out_dim, p.segs = p.batches = 1;
  p.bias[0] = a.bias;
  p.residual = a.residual, p.ldr = a.ldr;
  p.out[0] = a.y, p.ldo = a.ldy;
  p.save[0] = a.preact, p.lds = a.ldz;
  p.act = a.activation;
  p.status = a.status;
  const size_t size = elem_bytes(a.storage);
  p.vec = std::min(access_width(a.y, a.ldy, size), access_width(a.preact, a.ldz, size));
  p.bias_vec = aligned16(a.bias, 0, size);
  return forward(a.storage, g, &x, &w, nullptr, arena, guard, s);
}

extern "C" xvec_gpu_status xvec_gpu_gated_device(const xvec_gpu_gated_args* args) {
  xvec_gpu_status st = check_shape(args);
  if (st) return st;
  xvec_gpu_gated_args a = *args;
  if (!a.gate_weight || !a.up_weight || (a.n && (!a.x || !a.h)))
    return invalid("x, gate_weight, up_weight and h are required");
  if (!a.gate != !a.up) return invalid("gate and up are given together or not at all");
  Check c(elem_bytes(a.storage));
  c.ld("x", a.x, a.n, a.in_dim, &a.ldx);
  c.ld("the weights", a.gate_weight, a.out_dim, a.in_dim, &a.ldw);
  c.ld("h", a.h, a.n, a.out_dim, &a.ldh);
  c.ld("gate and up", a.gate, a.n, a.out_dim, &a.ldg);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("gate_weight", a.gate_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("up_weight", a.up_weight, a.out_dim, a.in_dim, a.ldw);
  c.in("gate_bias", a.gate_bias, 1, a.out_dim, a.out_dim);
  c.in("up_bias", a.up_bias, 1, a.out_dim, a.out_dim);
  c.out("h", a.h, a.n, a.out_dim, a.ldh);
  c.out("gate", a.gate, a.n, a.out_dim, a.ldg);
  c.out("up", a.up, a.n, a.out_dim, a.ldg);
  c.status(a.status);
  if ((st = c.overlaps())) return st;
  if (a.n == 0) return XVEC_GPU_OK;
  DeviceGuard guard;
  if ((st = guard.set(a.device))) return st;
  cudaStream_t s = static_cast<cudaStream_t>(a.stream);
  if (use_few_rows(a.storage, a.n, a.in_dim, a.out_dim, 2)) {
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
  Arena arena;
  Operand x = plan_operand(a.storage, a.x, a.n, a.in_dim, a.ldx, &arena);
  Operand wg = plan_operand(a.storage, a.gate_weight, a.out_dim, a.in_dim, a.ldw, &arena);
  Operand wu = plan_operand(a.storage, a.up_weight, a.out_dim, a.in_dim, a.ldw, &arena);
  GemmParams& p = g.p;
  p.rows = a.n, p.cols = a.out_dim, p.segs = p.batches = 1;
  p.bias[0] = a.gate_bias, p.bias[1] = a.up_bias;
  p.out[0] = a.h, p.ldo = a.ldh;
  p.save[0] = a.gate, p.save[1] = a.up, p.lds = a.ldg;
  p.act = a.activation;
  p.status = a.status;
  const size_t size = elem_bytes(a.storage);
  p.vec = std::min({access_width(a.h, a.ldh, size), access_width(a.gate, a.ldg, size),
                    access_width(a.up, a.ldg, size)});
  p.bias_vec = aligned16(a.gate_bias, 0, size) && aligned16(a.up_bias, 0, size);
  return forward(a.storage, g, &x, &wg, &wu, arena, guard, s);
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

xvec_gpu_status run_backward(const Backward& b, const DeviceGuard& guard) {
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
  // The plan: operands, both products and their scratch.
  Arena arena;
  Operand w[2], x;
  if (b.dx)
    for (int i = 0; i < b.parts; ++i)
      w[i] = plan_operand(b.storage, b.w[i], b.out_dim, b.in_dim, b.ldw, &arena);
  if (b.dw[0] || b.dw[1]) x = plan_operand(b.storage, b.x, b.n, b.in_dim, b.ldx, &arena);
  // The pre-activation gradients as one operand of `parts` matrices.  dy itself
  // where no activation changes it and it can be read in place.
  GemmOperand grad;
  grad.inner = b.out_dim, grad.outer = b.n;
  const bool direct = b.parts == 1 && b.act == XVEC_ACT_NONE && size == 2 &&
                      aligned16(b.dy, b.lddy, size);
  size_t grad_at = 0;
  if (direct) {
    grad.p = b.dy, grad.ld = b.lddy;
  } else {
    grad.ld = round8(b.out_dim);
    grad.plane = b.n * grad.ld;
    grad.planes = planes_of(b.storage) * b.parts;
    if (products) grad_at = arena.add((size_t)grad.planes * grad.plane * 2);
  }
  Slopes a{};
  a.dy = b.dy, a.z = b.pre[0], a.u = b.parts == 2 ? b.pre[1] : nullptr;
  a.lddy = b.lddy, a.ldz = b.ldpre, a.n = b.n, a.m = b.out_dim, a.act = b.act;
  a.ld = grad.ld;
  plan_slopes(&a);
  const bool scaled = b.storage == XVEC_STORAGE_FP16 && !direct && products;
  const size_t peaks_at = scaled ? arena.add((size_t)a.cols * a.chunks * 4) : 0;
  const size_t scale_at = scaled ? arena.add(4) : 0;
  const size_t sums_at = sums ? arena.add((size_t)2 * a.chunks * a.m * 4) : 0;
  GemmCall dx, dw;
  dx.mode = kDx;
  dx.depth = b.out_dim;
  dx.p.rows = b.n, dx.p.cols = b.in_dim, dx.p.segs = b.parts, dx.p.batches = 1;
  dx.p.out[0] = b.dx, dx.p.ldo = b.lddx;
  dx.p.vec = access_width(b.dx, b.lddx, size);
  dx.p.status = b.status;
  dw.mode = kDw;
  dw.depth = b.n;
  dw.p.rows = b.out_dim, dw.p.cols = b.in_dim, dw.p.segs = 1;
  dw.p.vec = 16;
  dw.p.ldo = b.lddw;
  dw.p.status = b.status;
  const int first = b.dw[0] ? 0 : 1;  // 1: only the second weight's gradient
  for (int i = first; i < b.parts && b.dw[i]; ++i) {
    dw.p.out[dw.p.batches++] = b.dw[i];
    dw.p.vec = std::min(dw.p.vec, access_width(b.dw[i], b.lddw, size));
  }
  if (b.dx && (st = plan_gemm(b.storage, &dx))) return st;
  if (dw.p.batches && (st = plan_gemm(b.storage, &dw))) return st;
  const size_t dx_partial = arena.add(dx.partial_bytes), dw_partial = arena.add(dw.partial_bytes);
  const size_t dx_runs = arena.add(dx.run_bytes), dw_runs = arena.add(dw.run_bytes);

  if ((st = arena.alloc(guard, s))) return st;
  Packs packs;
  for (Operand* o : {&w[0], &w[1], &x}) place(o, arena, &packs);
  if (!direct && products) grad.p = a.out = static_cast<uint16_t*>(arena.at(grad_at));
  if (sums) a.partial = static_cast<float*>(arena.at(sums_at));
  if (scaled) {
    a.peaks = static_cast<float*>(arena.at(peaks_at));
    dx.p.scale = dw.p.scale = a.scale = static_cast<float*>(arena.at(scale_at));
  }
  // Small packings share the gradient pass's launch; large ones want the warps that
  // its registers leave no room for (75103 x 402 fp32: 122 us together).
  int64_t packed = 0;
  for (int i = 0; i < packs.n; ++i) packed += packs.p[i].rows * packs.p[i].ld;
  const bool together = !direct && packed < 4'000'000;
  if (together) a.packs = packs;
  if (!direct && (st = slopes(b.storage, a, s))) return st;
  if (direct && sums && (st = chunk_sums(b.storage, a, s))) return st;
  if (!together && (st = run_packs(b.storage, packs, s))) return st;
  GemmParams& carrier = b.dx ? dx.p : dw.p;  // takes the column sums along
  if (sums) {
    carrier.sums = a.partial, carrier.sum_chunks = a.chunks, carrier.sum_cols = a.m;
    carrier.sum_out[0] = b.db[0], carrier.sum_out[1] = b.db[1];
    if (!products) return sum_columns(b.storage, carrier, s);
  }
  if (b.dx) {
    dx.a = grad;
    dx.b[0] = w[0].g, dx.b[1] = w[1].g;
    if (dx.partial_bytes) dx.p.partial = static_cast<float*>(arena.at(dx_partial));
    if (dx.run_bytes) dx.p.runs = static_cast<float*>(arena.at(dx_runs));
    if ((st = gemm(b.storage, dx, s))) return st;
  }
  if (dw.p.batches) {
    dw.a = grad;
    if (first) {
      dw.a.p = static_cast<const uint16_t*>(grad.p) + planes_of(b.storage) * grad.plane;
      dw.a.planes = planes_of(b.storage);
    }
    dw.b[0] = x.g;
    if (dw.partial_bytes) dw.p.partial = static_cast<float*>(arena.at(dw_partial));
    if (dw.run_bytes) dw.p.runs = static_cast<float*>(arena.at(dw_runs));
    // Directly after dx's product, whose inputs were complete when it began.
    dw.p.beside = b.dx && !dx.partial_bytes;
    if ((st = gemm(b.storage, dw, s))) return st;
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
  c.ld("dy", a.dy, a.n, a.out_dim, &a.lddy);
  c.ld("x", a.x, a.n, a.in_dim, &a.ldx);
  c.ld("weight", a.weight, a.out_dim, a.in_dim, &a.ldw);
  c.ld("preact", a.preact, a.n, a.out_dim, &a.ldz);
  c.ld("dx", a.dx, a.n, a.in_dim, &a.lddx);
  c.ld("dweight", a.dweight, a.out_dim, a.in_dim, &a.lddw);
  c.in("dy", a.dy, a.n, a.out_dim, a.lddy);
  c.in("x", a.x, a.n, a.in_dim, a.ldx);
  c.in("weight", a.weight, a.out_dim, a.in_dim, a.ldw);
  c.in("preact", a.preact, a.n, a.out_dim, a.ldz);
  c.out("dx", a.dx, a.n, a.in_dim, a.lddx);
  c.out("dweight", a.dweight, a.out_dim, a.in_dim, a.lddw);
  c.out("dbias", a.dbias, 1, a.out_dim, a.out_dim);
  c.status(a.status);
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
  return run_backward(b, guard);
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
  c.ld("dh", a.dh, a.n, a.out_dim, &a.lddh);
  c.ld("x", a.x, a.n, a.in_dim, &a.ldx);
  c.ld("the weights", a.gate_weight ? a.gate_weight : a.up_weight, a.out_dim, a.in_dim, &a.ldw);
  c.ld("gate and up", a.gate, a.n, a.out_dim, &a.ldg);
  c.ld("dx", a.dx, a.n, a.in_dim, &a.lddx);
  c.ld("the weight gradients", a.dgate_weight ? a.dgate_weight : a.dup_weight, a.out_dim,
       a.in_dim, &a.lddw);
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
  c.status(a.status);
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
  return run_backward(b, guard);
}

extern "C" xvec_gpu_status xvec_gpu_trim_scratch(int32_t device) {
  DeviceGuard guard;
  if (xvec_gpu_status st = guard.set(device)) return st;
  if (guard.pool) XVEC_CUDA(cudaMemPoolTrimTo(guard.pool, 0));
  return XVEC_GPU_OK;
}
