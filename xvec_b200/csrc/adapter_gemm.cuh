// adapter_gemm.cuh — the learned adapter's products on the tensor cores.
//
// Every product of the adapter is D [rows][cols] = sum over depth of A x B with
// its own operand order and epilogue (adapter.cuh, Mode):
//   kLinear  x W'            A and B contiguous along depth
//   kGated   x Wg', x Wu'    the same, two B's in one tile's two column halves
//   kDx      dz W            A contiguous along depth, B along the columns
//   kDw      dz' x           A contiguous along the rows, B along the columns
// so no operand is ever transposed in memory: the matrix instruction reads
// either order from shared memory.
//
//   CTA = 12 warps, persistent over tiles, one CTA per SM:
//     warp 0     TMA producer: 64 deep blocks of A (128 rows) and B into a ring of
//                stages (128-byte swizzle)
//     warp 1     tensor memory; one thread issues tcgen05.mma (fp32 accumulators,
//                two of them, so that a tile's epilogue overlaps the next tile)
//     warps 2-3  column sums of an earlier launch, where the call has some
//     warps 4-11 epilogue: tcgen05.ld, bias, activation, product, residual
//   PAIR: two CTAs on neighbouring SMs (cta_group::2) share a tile of 256 rows x
//   BN columns: each loads half of A's rows and half of B's columns and holds half
//   of the rows' sums.  Operands come out of shared memory at 64 bytes a clock: an
//   instruction of depth 16 reads 4 KB of A and BN x 16 bytes of B in each SM of a
//   pair, so 128 clocks for 256 columns (the matrix rate) and 96 for 128; a single
//   CTA's 128 x 128 reads 8 KB, 128 clocks for a quarter of the first's work, but it
//   starts and ends 1.5 us sooner, which decides for the smallest products.
//
// 16-bit storage multiplies its elements as they are.  float32 storage comes
// as three bfloat16 planes h + m + l (24 bits, x exactly); a stage holds one
// plane of A and of B, and the six products hh, hm, mh, mm, hl, lh are issued
// (what is left out is below 2^-24 of the product).  The accumulator's own
// additions truncate (measured: 48 of them leave 1.1e-6 of the 2-norm at depth
// 960), so hh has an accumulator of its own that leaves tensor memory every
// kRound blocks to be added in registers (8 truncations; 32 in a tile's first
// round), and the five products that are 2^8 times smaller have another that leaves
// at the end.  hh is drained while the small products of the same block are issued,
// so one accumulator of each suffices and the tile can keep 256 columns.  The planes come
// in the order m, h, l: m's stage is free after two thirds of the products, and the
// next block's first copy starts that much sooner (the ring holds two blocks).
// The drained sums take the registers that the other warps give up (setmaxnreg).
//
// LONG: sums of more than kRun blocks (2048 terms, float32 4096) are taken in runs of
// that many, each in fresh accumulators.  Truncation always points to zero: over 131072 terms of
// one sign a single 16-bit accumulator lost 8.4e-4 of the sum (1e-7 for each of its
// 8192 additions; binary16's half step is 4.9e-4).  16-bit types then hold a
// tile's sums in registers, as float32 does, where the runs are added in float32
// (linear backward 16384 x 2048 -> 1024 bf16 118 -> 120 us with runs of 2048 or 4096 terms;
// 8192^3 bf16 732 -> 766 with 2048, 753 with 4096).
// float32's small products need runs as well (262144 terms of either sign: 3.7e-6 of
// the 2-norm without); its registers are added up in a scratch of the epilogue's own,
// each thread reading back what it wrote itself, so that no sum has many terms.
//
// Every mbarrier wait is bounded; on expiry the kernel sets *status, stops
// issuing work, drains its own copies and frees its tensor memory.
#pragma once

#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "adapter.cuh"
#include "tcgen05.cuh"

namespace xvec {
namespace adapter {

constexpr int kBM = 128;      // rows per CTA (TMEM lanes)
constexpr int kBK = 64;       // depth per stage: 128 bytes, one swizzle row
constexpr uint32_t kABytes = kBM * kBK * 2;
constexpr int kBand = 8;      // row tiles per band of the tile order
// Registers of a thread where sums are held: of the first four warps, and of the epilogue's
// (together no more than the launch's; the host checks).
constexpr int kFewRegs = 56;
template <typename T>
constexpr int kManyRegs = std::is_same<T, float>::value ? 224 : 216;
// float32: depth blocks per accumulation in tensor memory.  A tile's first one is
// longer: so far the product runs ahead while the tile before is finished.
constexpr int kFirstRound = 8, kRound = 2;
// Whether block `k` of a run begins an accumulation.
__host__ __device__ constexpr bool opens_round(int k) {
  return k == 0 || (k >= kFirstRound && (k - kFirstRound) % kRound == 0);
}

template <int MODE, typename T, bool PAIR, int BN, bool LONG>
struct GemmShape {
  // Two epilogue warps per TMEM lane quarter, one per half of the columns.  (Four
  // on 256 columns cost a stage of the ring and were slower: 131072 x 1024 -> 1024
  // fp16 with silu and residual 360 us against 336.)
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 128 + kEpiWarps * 32;
  static constexpr int kBRows = PAIR ? BN / 2 : BN;  // B columns loaded per CTA
  static constexpr uint32_t kBBytes = kBRows * kBK * 2;
  // A stage holds one plane of a depth block (float32), or two blocks (16-bit): a
  // stage's handshake takes its single threads about 350 clocks, one block's
  // instructions 512 or less.
  static constexpr int kUnits = std::is_same<T, float>::value ? 1 : 2;
  static constexpr int kRun = run_blocks(std::is_same<T, float>::value);
  static_assert(kRun % kUnits == 0, "a stage belongs to one run");
  static constexpr uint32_t kBlockBytes = kABytes + kBBytes;
  static constexpr uint32_t kStageBytes = kUnits * kBlockBytes;
  // Columns that an epilogue warp finishes at a time, and their staging block of 32
  // rows: 128 bytes a row where its columns come in 64s (or 32 float32), else 64.
  static constexpr int kOutCols = BN / 2 / (MODE == kGated ? 2 : 1);  // outputs of a warp
  // Sums are held in registers (else read from tensor memory as they are finished).
  static constexpr bool kHold = std::is_same<T, float>::value || LONG;
  static constexpr int kStep = sizeof(T) == 2 && !kHold && kOutCols % 64 == 0 ? 64 : 32;
  static constexpr int kRowBytes = kStep * sizeof(T);
  static constexpr uint32_t kEpiBytes = kEpiWarps * 32 * kRowBytes;
  static constexpr int kFit = (int)((232448 - 1024 - 512 - kEpiBytes) / kStageBytes);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kEpiBytes + 1024 + 512;
  static constexpr int kTmemCols = BN == 192 ? 512 : 2 * BN;  // two accumulators, a power of two
  static_assert(kStages * kUnits >= 6, "shared memory too small for the stage ring");
};

// --- barriers, operands, matrix instructions --------------------------------------
// The producer and the issuer are single threads whose instruction count can bound
// the rate of the ring (a block has 512 clocks or less), so addresses are
// 32-bit shared ones, descriptors are kept as sums, and the limit and the abort
// flag are looked at only after a failed try.  (With a generic wait, a division
// and an abort check for each block they took 780 clocks.)
__device__ __forceinline__ bool try_bar(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Bounded: false once limit_ns passed or another role of the CTA raised *abort.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const volatile int* abort,
                                         uint64_t limit_ns) {
  if (try_bar(bar, parity)) return true;
  const uint64_t start = tc::global_ns();
  for (;;) {
    if (try_bar(bar, parity)) return true;
    if (*abort || tc::global_ns() - start > limit_ns) return false;
  }
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// One box of a [plane][outer][inner] operand.  PAIR: it completes on the barrier at
// the cluster address `bar`, which may belong to the other CTA.
template <bool PAIR>
__device__ __forceinline__ void load_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int x,
                                         int y, int z) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Matrix descriptor of an operand tile in 128-byte swizzle, without its address
// (which is added in units of 16 bytes).
//   along depth (K-major): rows of 128 bytes, 8-row groups 1024 bytes apart;
//     16 deep = 32 bytes further.
//   along rows (MN-major): blocks of 64 rows x 64 deep (8 KB, the leading
//     offset), in a block 8-deep groups 1024 bytes apart; 16 deep = 2048 bytes
//     further.
template <bool MN>
constexpr uint64_t kTileDesc = ((uint64_t)(MN ? 8192 >> 4 : 1) << 16) |
                               ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
template <bool MN>
constexpr uint64_t kDepthStep = MN ? 2048 >> 4 : 32 >> 4;

template <bool PAIR>
__device__ __forceinline__ void mma_16bit(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t acc) {
  if constexpr (PAIR)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Arrives on the barrier at the shared-memory address `bar` of this CTA (PAIR: of both
// CTAs) once every MMA this thread issued so far has completed.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    tc::mma_commit<false>(bar);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

// --- epilogue input and output ------------------------------------------------------
// A warp holds 32 rows of values, one row per lane.  They reach memory (and a
// residual comes from it) through a staging block of 32 rows of RB bytes, so that
// each instruction covers whole row segments of RB bytes: RB / 16 lanes of 16
// bytes per row.  The 16-byte parts of a row are permuted by its number, which
// keeps both directions free of bank conflicts.
template <int RB>
__device__ __forceinline__ uint32_t stage_at(uint32_t buf, int row, int part) {
  return buf + row * RB + ((part ^ (RB == 128 ? row & 7 : (row >> 1) & 3)) << 4);
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  uint4 u;
  if constexpr (std::is_same<T, float>::value) {
    u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                   __float_as_uint(v[3]));
  } else {
    u = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                   pack2<T>(v[6], v[7]));
  }
  return u;
}

// The staging rows to memory in accesses of W bytes: 32 W / RB rows at a time.
template <typename T, int RB, int W>
__device__ __forceinline__ void copy_out(uint32_t buf, T* out, int64_t ld, int rows, int lane) {
  constexpr int kLanes = RB / W, kRows = 32 / kLanes;  // lanes of a row, rows at a time
  const int at = lane % kLanes * W, row = lane / kLanes;
  char* dst = reinterpret_cast<char*>(out) + at;
#pragma unroll
  for (int i0 = 0; i0 < 32 / kRows; i0 += 8) {
    uint32_t u[8][W / 4];
#pragma unroll
    for (int i = 0; i < 8 && i0 + i < 32 / kRows; ++i) {
      const uint32_t a = stage_at<RB>(buf, (i0 + i) * kRows + row, at / 16) + at % 16;
      if constexpr (W == 16) {
        const uint4 t = lds16(a);
        u[i][0] = t.x, u[i][1] = t.y, u[i][2] = t.z, u[i][3] = t.w;
      } else if constexpr (W == 8) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(u[i][0]), "=r"(u[i][1]) : "r"(a) : "memory");
      } else {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u[i][0]) : "r"(a) : "memory");
      }
    }
#pragma unroll
    for (int i = 0; i < 8 && i0 + i < 32 / kRows; ++i) {
      const int r = (i0 + i) * kRows + row;
      if (r >= rows) continue;
      char* p = dst + r * ld * (int)sizeof(T);
      if constexpr (W == 16)
        *reinterpret_cast<uint4*>(p) = make_uint4(u[i][0], u[i][1], u[i][2], u[i][3]);
      else if constexpr (W == 8)
        *reinterpret_cast<uint2*>(p) = make_uint2(u[i][0], u[i][1]);
      else
        *reinterpret_cast<uint32_t*>(p) = u[i][0];
    }
  }
}

// N values of this lane's row into the staging block, from part `part` on.
template <typename T, int RB, int N>
__device__ __forceinline__ void stage_put(uint32_t buf, int part, const float* v, int lane) {
  constexpr int kPart = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < N / kPart; ++c)
    sts16(stage_at<RB>(buf, lane, part + c), pack16<T>(v + c * kPart));
}
// The staging block to out[row * ld + column], rows and cols of it.  width: the
// bytes of an access that its rows allow (16, 8, 4; 2 for 16-bit types).
template <typename T, int RB>
__device__ __forceinline__ void stage_out(uint32_t buf, T* out, int64_t ld, int rows, int cols,
                                          int width, int lane) {
  constexpr int kPart = 16 / sizeof(T), kCols = RB / sizeof(T);
  __syncwarp();
  if (cols >= kCols && width >= 4) {
    if (width == 16) copy_out<T, RB, 16>(buf, out, ld, rows, lane);
    else if (width == 8) copy_out<T, RB, 8>(buf, out, ld, rows, lane);
    else copy_out<T, RB, 4>(buf, out, ld, rows, lane);
  } else {
    // A column a lane, a row after the other.
#pragma unroll
    for (int c0 = 0; c0 < kCols; c0 += 32) {
      const int col = c0 + lane;
      if (col < cols) {
#pragma unroll 8
        for (int r = 0; r < rows; ++r) {
          const uint32_t a = stage_at<RB>(buf, r, col / kPart) + (col % kPart) * sizeof(T);
          if constexpr (sizeof(T) == 4) {
            float f;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
            out[r * ld + col] = f;
          } else {
            uint16_t b;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(b) : "r"(a) : "memory");
            reinterpret_cast<uint16_t*>(out)[r * ld + col] = b;
          }
        }
      }
    }
  }
  __syncwarp();
}
// Writes v (this lane's row) to base[row * ld + column], a staging block at a time.
template <typename T, int RB, int N>
__device__ __forceinline__ void emit(uint32_t buf, T* base, int64_t ld, int rows, int cols, int width,
                                     const float (&v)[N], int lane) {
  constexpr int kCols = RB / sizeof(T);
  static_assert(N % kCols == 0, "whole staging rows");
#pragma unroll
  for (int h = 0; h < N / kCols; ++h) {
    stage_put<T, RB, kCols>(buf, 0, v + h * kCols, lane);
    stage_out<T, RB>(buf, base + h * kCols, ld, rows, cols - h * kCols, width, lane);
  }
}

// A block of 32 rows on its way in: requested early (start), added to this
// lane's row later (add).  Rows that do not start on 16 bytes come as the granules
// that hold them, one more than they have parts (each lane keeps its row's last),
// and are shifted together from the staging block.  Rows or columns that do not
// exist are not read.
template <typename T, int RB>
struct Incoming {
  static constexpr int kParts = RB / 16, kPart = 16 / sizeof(T), N = RB / sizeof(T);
  uint4 v[kParts], last;
  uint32_t off;  // of this lane's row

  __device__ __forceinline__ void start(const T* base, int64_t ld, int rows, int cols, int lane) {
    // Without columns the row's address may lie past the matrix, and the granule
    // that it falls into with it.
    if (cols <= 0) rows = 0;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int r = i * (32 / kParts) + lane / kParts;
      const uintptr_t p = (uintptr_t)(base + r * ld), end = (uintptr_t)(base + r * ld + cols);
      v[i] = granule(p / 16 * 16 + lane % kParts * 16, r < rows ? end : 0);
    }
    const uintptr_t p = (uintptr_t)(base + lane * ld), end = (uintptr_t)(base + lane * ld + cols);
    off = (uint32_t)p & 15;
    last = granule(p / 16 * 16 + RB, lane < rows && off ? end : 0);
  }
  __device__ __forceinline__ void add(uint32_t buf, float (&f)[N], int lane) {
#pragma unroll
    for (int i = 0; i < kParts; ++i)
      sts16(stage_at<RB>(buf, i * (32 / kParts) + lane / kParts, lane % kParts), v[i]);
    __syncwarp();
    uint4 u = lds16(stage_at<RB>(buf, lane, 0));
    const bool straight = __all_sync(0xffffffffu, off == 0);
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
      const uint4 next = c + 1 < kParts ? lds16(stage_at<RB>(buf, lane, c + 1)) : last;
      if (!straight) u = shifted<T>(u, next, off);
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < kPart; ++j) f[c * kPart + j] += to_f(t[j]);
      u = next;
    }
    __syncwarp();
  }
};

// x += the biases of its columns, `cols` of which exist (the same for all lanes).
template <typename T, int N>
__device__ __forceinline__ void add_bias(const T* bias, int cols, bool vec, float (&x)[N]) {
  if (!bias) return;
  if (vec && cols >= N) {
#pragma unroll
    for (int c = 0; c < N * (int)sizeof(T) / 16; ++c) {
      const uint4 u = reinterpret_cast<const uint4*>(bias)[c];
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[c * (16 / sizeof(T)) + j] += to_f(t[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < cols) x[j] += to_f(bias[j]);
  }
}

// --- the kernel ---------------------------------------------------------------
template <int MODE, typename T, bool PAIR, int BN, bool LONG>
__global__ void __launch_bounds__(GemmShape<MODE, T, PAIR, BN, LONG>::kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap0,
                const __grid_constant__ CUtensorMap bmap1, const __grid_constant__ GemmParams p) {
  using namespace tc;
  using S = GemmShape<MODE, T, PAIR, BN, LONG>;
  constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDx || MODE == kDw;
  constexpr int P = std::is_same<T, float>::value ? 3 : 1;  // planes
  constexpr int kStages = S::kStages, kEpiWarps = S::kEpiWarps;
  constexpr int kTileRows = PAIR ? 256 : 128;
  constexpr int kTileCols = MODE == kGated ? BN / 2 : BN;
  constexpr int kWarpCols = BN / 2;  // accumulator columns per epilogue warp
  constexpr int kOutCols = S::kOutCols, kStep = S::kStep, RB = S::kRowBytes;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = tiles + kStages * S::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + S::kEpiBytes);
  uint64_t* empty = full + kStages;   // the MMAs have read the stage
  uint64_t* tfull = empty + kStages;  // [2] accumulator ready (float32: hh, small)
  uint64_t* tempty = tfull + 2;       // [2] accumulator drained (issuing CTA's count)
  uint64_t* mdone = tempty + 2;       // all issued MMAs retired
  uint32_t* issued = reinterpret_cast<uint32_t*>(mdone + 1);  // [kStages] copies per stage
  uint32_t* units = issued + kStages;  // [kStages] blocks of the stage's last filling
  uint32_t* tmem_slot = units + kStages;
  __shared__ int s_abort_storage;
  volatile int* s_abort = &s_abort_storage;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const bool issuer = rank == 0;
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const int workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int tiles_mn = p.tiles_m * p.tiles_n;
  const int items = tiles_mn * p.batches * p.splits;
  const int all_blocks = p.segs * p.blocks;
  const uint64_t limit = p.wait_ns;
  auto fail = [&] {
    if (p.status) atomicExch(p.status, (int)XVEC_GPU_TIMEOUT);
    *s_abort = 1;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      issued[s] = units[s] = 0;
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (PAIR ? 2 : 1) * kEpiWarps);
    }
    mbar_init(mdone, 1);
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "n"(S::kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "n"(S::kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tmem_fence_before();
  }
  if (p.beside) pdl_launch();  // (all it reads comes through TMA, from L2)
  else pdl_begin();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tmem_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Work item -> split, batch, tile.  Tiles go down bands of kBand row tiles, so
  // that those running at a time share both A's rows and B's columns in L2.
  struct Item {
    int batch, tm, tn, k0, k1, split;
  };
  auto item_of = [&](int i) {
    Item it;
    const int t = i % tiles_mn, g = i / tiles_mn;
    it.batch = g % p.batches;
    it.split = g / p.batches;
    const int band = t / (kBand * p.tiles_n), in = t - band * kBand * p.tiles_n;
    const int height = min(kBand, p.tiles_m - band * kBand);
    it.tn = in / height;
    it.tm = band * kBand + in - it.tn * height;
    it.k0 = it.split * p.blocks_per_split;
    it.k1 = min(all_blocks, it.k0 + p.blocks_per_split);
    return it;
  };

  // Held sums: 384 threads of 168 registers become 128 of kFewRegs and 256 of kManyRegs.
  if (warp < 4) {
    if constexpr (S::kHold) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer ----------------
      const uint32_t tiles_at = smem_u32(tiles), empty_at = smem_u32(empty);
      const uint32_t full_at = smem_u32(full), bars = PAIR ? cluster_addr(full, 0) : full_at;
      uint32_t stage = 0, phase = 0, count = 0;  // count: stages filled
      bool ok = true;
      for (int i = worker; i < items && ok; i += workers) {
        const Item it = item_of(i);
        const int row0 = it.tm * kTileRows + (int)rank * kBM;
        const int col0 = it.tn * kTileCols + (MODE == kGated ? 0 : (int)rank * S::kBRows);
        int seg = it.k0 / p.blocks;
        int k = (it.k0 - seg * p.blocks) * kBK;
        const int k_end = p.blocks * kBK;
        // One block of A and B into `a`, from depth k of product seg, plane pl.
        auto load = [&](uint32_t bar, uint32_t a, int pl) {
          const uint32_t b = a + kABytes;
          const int az = (MODE == kDw ? it.batch : MODE == kDx ? seg : 0) * P + pl;
          const CUtensorMap* bm = (MODE == kDx && seg) || (MODE == kGated && PAIR && rank) ? &bmap1
                                                                                          : &bmap0;
          if constexpr (A_MN) {
            load_box<PAIR>(&amap, bar, a, row0, k, az);
            load_box<PAIR>(&amap, bar, a + 8192, row0 + 64, k, az);
          } else {
            load_box<PAIR>(&amap, bar, a, k, row0, az);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int c = 0; c < S::kBRows / 64; ++c)
              load_box<PAIR>(bm, bar, b + c * 8192, col0 + c * 64, k, pl);
          } else {
            // Gated: the gate's columns, then the up's (PAIR: one in each CTA).
            load_box<PAIR>(bm, bar, b, k, col0, pl);
            if constexpr (MODE == kGated && !PAIR)
              load_box<PAIR>(&bmap1, bar, b + S::kBBytes / 2, k, col0, pl);
          }
        };
        for (int n = it.k1 - it.k0; n > 0 && ok; n -= S::kUnits) {
#pragma unroll
          for (int pl = 0; pl < P; ++pl) {
            if (!(ok = ok && wait_bar(empty_at + stage * 8, phase ^ 1, s_abort, limit))) break;
            const uint32_t at = tiles_at + stage * S::kStageBytes, bar = bars + stage * 8;
            const uint32_t blocks = min(n, S::kUnits);
            if (issuer) expect_bytes(full_at + stage * 8, (PAIR ? 2 : 1) * blocks * S::kBlockBytes);
            load(bar, at, P == 1 ? 0 : pl == 0 ? 1 : pl == 1 ? 0 : 2);
            if constexpr (P == 1) {
              if ((k += kBK) == k_end) k = 0, ++seg;
              if (blocks > 1) {
                load(bar, at + S::kBlockBytes, pl);
                if ((k += kBK) == k_end) k = 0, ++seg;
              }
            }
            units[stage] = blocks;
            ++count;
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
          if (P == 3 && (k += kBK) == k_end) k = 0, ++seg;
        }
      }
      if (!ok) fail();
      for (uint32_t s = 0; s < kStages; ++s)
        issued[s] = count / kStages + (s < count % kStages ? 1 : 0);
    } else if (warp == 1 && lane == 0 && issuer) {
      // ---------------- MMA issuer ----------------
      const uint32_t full_at = smem_u32(full), empty_at = smem_u32(empty);
      const uint32_t tfull_at = smem_u32(tfull), tempty_at = smem_u32(tempty);
      const uint64_t a0 = kTileDesc<A_MN> + (smem_u32(tiles) >> 4);
      const uint64_t b0 = kTileDesc<B_MN> + ((smem_u32(tiles) + kABytes) >> 4);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      // Waits for the next stage; its number.
      auto next = [&](uint32_t* at) {
        *at = stage;
        const bool got = wait_bar(full_at + stage * 8, phase, s_abort, limit);
        if (++stage == kStages) stage = 0, phase ^= 1;
        tmem_fence_after();
        return got;
      };
      // A's block in stage i times B's in stage j, both `off` further, into d; keep = 0
      // overwrites it.
      auto multiply = [&](uint32_t i, uint32_t j, uint32_t d, uint32_t keep, uint32_t off = 0) {
        const uint64_t a = a0 + (i * (S::kStageBytes >> 4) + off);
        const uint64_t b = b0 + (j * (S::kStageBytes >> 4) + off);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_16bit<PAIR>(d, a + k * kDepthStep<A_MN>, b + k * kDepthStep<B_MN>, p.idesc,
                          k == 0 ? keep : 1u);
      };
      uint32_t round = 0, run = 0;
      // The product of blocks [k0, k1), one run (or a whole tile).
      auto multiply_run = [&](int k0, int k1) {
        if constexpr (P == 1) {
          const uint32_t acc = run & 1, d = tmem_base + acc * BN;
          if (!(ok = wait_bar(tempty_at + acc * 8, ((run >> 1) & 1) ^ 1, s_abort, limit))) return;
          tmem_fence_after();
          for (int k = k0; k < k1; k += S::kUnits) {
            uint32_t at;
            if (!(ok = next(&at))) break;
            multiply(at, at, d, k > k0);
            if (k + 1 < k1) multiply(at, at, d, 1, S::kBlockBytes >> 4);
            commit<PAIR>(empty_at + at * 8);
          }
          commit<PAIR>(tfull_at + acc * 8);
        } else {
          const uint32_t d = tmem_base, small = tmem_base + BN;
          for (int k = k0; k < k1; ++k) {
            const bool opens = opens_round(k - k0);
            const bool closes = k + 1 == k1 || opens_round(k + 1 - k0);
            uint32_t h, m, l;
            if (k == k0 && !(ok = wait_bar(tempty_at + 8, (run & 1) ^ 1, s_abort, limit))) break;
            if (!(ok = next(&m))) break;
            multiply(m, m, small, k > k0);
            if (opens) {
              if (!(ok = wait_bar(tempty_at, (round & 1) ^ 1, s_abort, limit))) break;
              tmem_fence_after();
              ++round;
            }
            if (!(ok = next(&h))) break;
            multiply(h, h, d, !opens);
            if (closes) commit<PAIR>(tfull_at);
            multiply(h, m, small, 1);
            multiply(m, h, small, 1);
            commit<PAIR>(empty_at + m * 8);
            if (!(ok = next(&l))) break;
            multiply(h, l, small, 1);
            multiply(l, h, small, 1);
            commit<PAIR>(empty_at + h * 8);
            commit<PAIR>(empty_at + l * 8);
          }
          commit<PAIR>(tfull_at + 8);
        }
      };
      for (int i = worker; i < items && ok; i += workers) {
        const Item it = item_of(i);
        if constexpr (LONG) {
          for (int k = it.k0; k < it.k1 && ok; k += S::kRun, ++run)
            multiply_run(k, min(it.k1, k + S::kRun));
        } else {
          multiply_run(it.k0, it.k1);
          ++run;
        }
      }
      if (!ok) fail();
      // Retire every issued MMA before tensor memory is released.
      mma_commit<PAIR>(smem_u32(mdone));
      if (!mbar_wait(mdone, 0, nullptr)) fail();
    } else if (warp >= 2 && p.sums) {
      column_sums<T>(p.sums, p.sum_chunks, p.sum_cols, p.sum_out[0], p.sum_out[1],
                     (int)blockIdx.x * 2 + warp - 2, (int)gridDim.x * 2, lane);
    }
  } else {
    // ---------------- epilogue ----------------
    if constexpr (S::kHold)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs<T>));
    const int quarter = warp & 3, ew = warp - 4, group = ew >> 2;
    const uint32_t buf = smem_u32(staging + ew * 32 * RB);
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tfull_at = smem_u32(tfull);
    // Waits for accumulator `acc`.  One lane polls; the others wait at the shuffle.
    auto wait_acc = [&](uint32_t acc, uint32_t parity) {
      int ok = 1;
      if (lane == 0 && !wait_bar(tfull_at + acc * 8, parity, s_abort, limit)) {
        fail();
        ok = 0;
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      tmem_fence_after();
      return ok != 0;
    };
    auto release_acc = [&](uint32_t acc) {
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_remote(cluster_addr(&tempty[acc], 0));
        else mbar_arrive(&tempty[acc]);
      }
    };
    // Accumulator column of output column c of the warp (which: the gate's or the
    // up's sums).
    auto acc_col = [&](int which, int c) {
      return which * (BN / 2) + group * kOutCols + c;
    };
    using Step = float[S::kStep];
    auto limit32 = [](int64_t c) { return (int)max((int64_t)0, min((int64_t)kStep, c)); };
    // float32: this thread's sums of the finished runs, a warp's 32 lanes side by side.
    // (The address is not kept in registers, of which none are left.)
    auto runs = [&](int at) {
      return p.runs + (((int64_t)blockIdx.x * kEpiWarps + ew) * kWarpCols + at) * 32 + lane;
    };
    // (From L2: this launch may have begun before it waited for any other, p.beside.)
    constexpr bool kScaled = std::is_same<T, __half>::value && (MODE == kDx || MODE == kDw);
    const float scale = kScaled && p.scale ? __ldcg(p.scale) : 1.f;
    uint32_t round = 0, run = 0;
    int done = 0;  // blocks of item i whose sums are in scratch (float32, LONG)
    for (int i = worker; i < items;) {
      const Item it = item_of(i);
      const int64_t row0 = (int64_t)it.tm * kTileRows + rank * kBM + quarter * 32;
      const int rows = (int)max((int64_t)0, min((int64_t)32, p.rows - row0));
      const int64_t warp_col = (int64_t)it.tn * kTileCols + group * kOutCols;
      const int64_t cols = p.cols - warp_col;  // from the warp's first one (may be negative)
      const T* res = MODE == kLinear && p.splits == 1 && p.residual
                         ? static_cast<const T*>(p.residual) + row0 * p.ldr + warp_col
                         : nullptr;
      Incoming<T, RB> in;
      // (Held sums leave no registers for it.)
      if (MODE == kLinear && !S::kHold && res) in.start(res, p.ldr, rows, limit32(cols), lane);
      // Finishes kStep columns from `at` on: v the sums (gated: the gate's; up(h, u)
      // then gives the up's, 32 at a time, since not all are held at once).
      auto finish = [&](int at, Step& v, auto&& up) {
        const int n = limit32(cols - at);
        const int64_t col = warp_col + at;
        if (p.splits > 1) {
          constexpr int kPlanes = MODE == kGated ? 2 : 1;
          float* dst = p.partial +
                       ((int64_t)(it.split * p.batches + it.batch) * kPlanes * p.rows + row0) *
                           p.ldp + col;
          // (ldp covers whole steps.)
          if (n > 0) emit<float, RB>(buf, dst, p.ldp, rows, kStep, 16, v, lane);
          if constexpr (MODE == kGated) {
#pragma unroll
            for (int h = 0; h < kStep / 32; ++h) {
              float u[32];
              up(h, u);
              if (n > 0)
                emit<float, RB>(buf, dst + p.rows * p.ldp + h * 32, p.ldp, rows, 32, 16, u, lane);
            }
          }
          return;
        }
        if (MODE == kLinear && S::kHold && res) in.start(res + at, p.ldr, rows, n, lane);
        [[maybe_unused]] const bool vec = p.bias_vec != 0;  // (forward products)
        auto biases = [&](int which) {
          const T* b = static_cast<const T*>(p.bias[which]);
          return b ? b + col : b;
        };
        auto saved = [&](int which) {
          return static_cast<T*>(p.save[which]) + row0 * p.lds + col;
        };
        if constexpr (MODE == kLinear || MODE == kGated) {
          add_bias(biases(0), n, vec, v);
          if (p.save[0] && n > 0) emit<T, RB>(buf, saved(0), p.lds, rows, n, p.vec, v, lane);
          activate_all<T>(p.act, v);
        }
        if constexpr (MODE == kGated) {
#pragma unroll
          for (int h = 0; h < kStep / 32; ++h) {
            float u[32];
            up(h, u);
            const T* b = biases(1);
            add_bias(b ? b + h * 32 : b, n - h * 32, vec, u);
            if (p.save[1]) stage_put<T, RB, 32>(buf, h * 32 * (int)sizeof(T) / 16, u, lane);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[h * 32 + j] *= u[j];
          }
          if (p.save[1]) stage_out<T, RB>(buf, saved(1), p.lds, rows, n, p.vec, lane);
        }
        if constexpr (kScaled) {
#pragma unroll
          for (int j = 0; j < kStep; ++j) v[j] *= scale;
        }
        if (MODE == kLinear && res && n > 0) {
          in.add(buf, v, lane);
          if (!S::kHold && at + kStep < kOutCols)
            in.start(res + at + kStep, p.ldr, rows, limit32(cols - at - kStep), lane);
        }
        if (n > 0)
          emit<T, RB>(buf, static_cast<T*>(p.out[MODE == kDw ? it.batch : 0]) + row0 * p.ldo + col,
                      p.ldo, rows, n, p.vec, v, lane);
      };
      if constexpr (!S::kHold) {
        const uint32_t acc = run & 1, t = tmem_base + acc * BN + lanes;
        if (!wait_acc(acc, (run >> 1) & 1)) break;
        ++run;
        // N sums; the accumulator is freed with its last ones.
        auto take = [&](int which, int at, auto& v) {
          constexpr int N = sizeof(v) / 4;
          uint32_t raw[N / 32][32];
#pragma unroll
          for (int c = 0; c < N / 32; ++c) tmem_ld32(t + acc_col(which, at + c * 32), raw[c]);
          tmem_wait_ld();
          if (which == (MODE == kGated ? 1 : 0) && at + N == kOutCols) release_acc(acc);
#pragma unroll
          for (int c = 0; c < N / 32; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) v[c * 32 + j] = __uint_as_float(raw[c][j]);
        };
#pragma unroll 1
        for (int at = 0; at < kOutCols; at += kStep) {
          Step v;
          take(0, at, v);
          finish(at, v, [&](int h, float (&u)[32]) { take(1, at + h * 32, u); });
        }
      } else {
        // 32 sums at a time: the output columns' (gated: a gate's 32, then the up's).
        constexpr int kSums = kWarpCols / 32, kPer = MODE == kGated ? 2 : 1;
        float sum[kSums][32];
        auto drain = [&](uint32_t t, bool first) {
#pragma unroll
          for (int c = 0; c < 2 * kSums; ++c) {
            uint32_t raw[16];
            tmem_ld16(t + lanes + acc_col((c >> 1) % kPer, (c >> 1) / kPer * 32) + (c & 1) * 16, raw);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float& f = sum[c >> 1][(c & 1) * 16 + j];
              f = first ? __uint_as_float(raw[j]) : f + __uint_as_float(raw[j]);
            }
          }
        };
        bool ok = true;
        if constexpr (P == 1) {
          for (int k = it.k0; k < it.k1 && ok; k += S::kRun, ++run) {
            const uint32_t acc = run & 1;
            if (!(ok = wait_acc(acc, (run >> 1) & 1))) break;
            drain(tmem_base + acc * BN, k == it.k0);
            release_acc(acc);
          }
        } else {
          const int k0 = LONG ? it.k0 + done : it.k0;
          const int k1 = LONG ? min(it.k1, k0 + S::kRun) : it.k1;
          for (int k = k0; k < k1 && ok; k += k == k0 ? kFirstRound : kRound, ++round) {
            if (!(ok = wait_acc(0, round & 1))) break;
            drain(tmem_base, k == k0);
            release_acc(0);
          }
          if (ok && (ok = wait_acc(1, run & 1))) {
            drain(tmem_base + BN, false);
            release_acc(1);
          }
          ++run;
          if constexpr (LONG) {
            if (ok && done) {
              const float* r = runs(0);
#pragma unroll
              for (int j = 0; j < kWarpCols; ++j) {
                sum[j / 32][j % 32] += r[j * 32];
                if (j % 8 == 7) asm volatile("" ::: "memory");  // (eight on their way)
              }
            }
            if (ok && k1 < it.k1) {
              float* r = runs(0);
#pragma unroll
              for (int j = 0; j < kWarpCols; ++j) r[j * 32] = sum[j / 32][j % 32];
              done += S::kRun;
              continue;
            }
          }
        }
        if (!ok) break;
        // A rolled loop over steps that always takes the first sums and moves the
        // others up: unrolled, its addresses alone made the sums spill.
#pragma unroll 1
        for (int at = 0; at < kOutCols; at += kStep) {
          finish(at, sum[0], [&](int, float (&u)[32]) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] = sum[kPer - 1][j];
          });
#pragma unroll
          for (int i = 0; i + kPer < kSums; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[i][j] = sum[i + kPer][j];
        }
      }
      done = 0;
      i += workers;
    }
  }

  __syncthreads();
  // Drain: every copy either CTA issued has landed before either leaves
  // (already true unless a role gave up).  The first CTA's barriers count
  // both CTAs' copies; a stage phase that the second CTA issued but the first
  // never armed is armed here for its half.
  if constexpr (PAIR) cluster_sync_all();
  if (threadIdx.x == 0 && issuer) {
    for (int s = 0; s < kStages; ++s) {
      const uint32_t mine = issued[s];
      const uint32_t other = PAIR ? ld_cluster_u32(cluster_addr(&issued[s], 1)) : mine;
      // Where the second CTA gave up before the first, its half never comes: the
      // wait then only gives the first's own copies ample time.
      if (mine > 0 &&
          !mbar_wait(&full[s], (mine - 1) & 1, nullptr, other < mine ? 20000000ull : kWaitLimitNs))
        fail();
      if (PAIR && other > mine) {
        mbar_expect_tx(&full[s], ld_cluster_u32(cluster_addr(&units[s], 1)) * S::kBlockBytes);
        if (!mbar_wait(&full[s], mine & 1, nullptr)) fail();
      }
    }
  }
  if (p.beside) pdl_wait();
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tmem_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "n"(S::kTmemCols));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "n"(S::kTmemCols));
  }
}

// --- split sums ------------------------------------------------------------------
// Adds the splits' partial sums in their order and finishes as the kernel would.
template <int MODE, typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ GemmParams p) {
  pdl_begin();
  const int64_t groups = (p.cols + 3) / 4;
  const int64_t total = groups * p.rows;
  const int batch = blockIdx.y;
  constexpr int kPlanes = MODE == kGated ? 2 : 1;
  const int64_t step = (int64_t)p.batches * kPlanes * p.rows * p.ldp;  // between splits
  const float scale = p.scale ? *p.scale : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / groups, col = (i - row * groups) * 4;
    float v[kPlanes][4] = {};
#pragma unroll
    for (int h = 0; h < kPlanes; ++h) {
      const float* src = p.partial + ((int64_t)(batch * kPlanes + h) * p.rows + row) * p.ldp + col;
      for (int s = 0; s < p.splits; ++s) {
        const float4 t = *reinterpret_cast<const float4*>(src + s * step);
        v[h][0] += t.x, v[h][1] += t.y, v[h][2] += t.z, v[h][3] += t.w;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = col + j;
      if (c >= p.cols) break;
      float y = v[0][j] * scale;
      if (MODE == kLinear || MODE == kGated) {
        if (p.bias[0]) y += to_f(static_cast<const T*>(p.bias[0])[c]);
        if (p.save[0]) static_cast<T*>(p.save[0])[row * p.lds + c] = from_f<T>(y);
        y = activate<T>(p.act, y);
      }
      if constexpr (MODE == kGated) {
        float u = v[1][j];
        if (p.bias[1]) u += to_f(static_cast<const T*>(p.bias[1])[c]);
        if (p.save[1]) static_cast<T*>(p.save[1])[row * p.lds + c] = from_f<T>(u);
        y *= u;
      }
      if (MODE == kLinear && p.residual) y += to_f(static_cast<const T*>(p.residual)[row * p.ldr + c]);
      static_cast<T*>(p.out[batch])[row * p.ldo + c] = from_f<T>(y);
    }
  }
}

// --- host side -----------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static const auto fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// The operand as [planes][outer][inner] 16-bit elements, boxes of [box_outer][64].
inline bool operand_map(CUtensorMap* map, const GemmOperand& o, int box_outer) {
  auto fn = encode_tiled();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer, (cuuint64_t)o.planes};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.ld) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_outer, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(o.p), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, typename T, bool PAIR, int BN, bool LONG>
xvec_gpu_status launch_sums(const GemmCall& c, cudaStream_t s) {
  GemmParams p = c.p;
  using S = GemmShape<MODE, T, PAIR, BN, LONG>;
  constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDx || MODE == kDw;
  CUtensorMap a, b0, b1;
  const int b_box = B_MN ? kBK : (MODE == kGated && !PAIR) ? S::kBRows / 2 : S::kBRows;
  if (!operand_map(&a, c.a, A_MN ? kBK : kBM) || !operand_map(&b0, c.b[0], b_box) ||
      !operand_map(&b1, c.b[1].p ? c.b[1] : c.b[0], b_box)) {
    set_error("adapter: no tensor map for an operand");
    return XVEC_GPU_CUDA_ERROR;
  }
  // Accumulator float32, operands binary16 (0) or bfloat16 (1), their orders, N, M.
  const uint32_t f = c.bf16 ? 1u : 0u;
  p.idesc = (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
            ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
  auto kern = gemm_kernel<MODE, T, PAIR, BN, LONG>;
  static std::atomic<uint64_t> ready{0};  // by device
  const uint64_t bit = 1ull << (c.device & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    XVEC_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)S::kSmemBytes));
    if (S::kHold) {
      // The register split needs the whole block's share at launch, or it would wait.
      cudaFuncAttributes fa;
      XVEC_CUDA(cudaFuncGetAttributes(&fa, kern));
      if (fa.numRegs * S::kThreads < 128 * kFewRegs + (S::kThreads - 128) * kManyRegs<T>) {
        set_error("adapter: the matrix kernel was built with %d registers", fa.numRegs);
        return XVEC_GPU_UNSUPPORTED;
      }
    }
    if (c.device < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.batches * p.splits;
  const int sms = c.sms;
  const int64_t ctas = PAIR ? std::min<int64_t>(items, sms / 2) * 2 : std::min<int64_t>(items, sms);
  XVEC_CUDA(launch_pdl(kern, dim3((unsigned)ctas), S::kThreads, S::kSmemBytes, s,
                       PAIR ? 2 : 1, a, b0, b1, p));
  if (p.splits > 1) {
    const int64_t groups = (p.cols + 3) / 4 * p.rows;
    XVEC_CUDA(launch_pdl(finish_kernel<MODE, T>,
                         dim3((unsigned)std::min<int64_t>((groups + 255) / 256, 1184),
                              (unsigned)p.batches),
                         256, 0, s, 1, p));
  }
  return XVEC_GPU_OK;
}

template <int MODE, typename T, bool PAIR, int BN>
xvec_gpu_status launch_shape(const GemmCall& c, cudaStream_t s) {
  const bool many = c.p.blocks_per_split > run_blocks(std::is_same<T, float>::value);
  return many ? launch_sums<MODE, T, PAIR, BN, true>(c, s)
              : launch_sums<MODE, T, PAIR, BN, false>(c, s);
}

template <int MODE, typename T>
xvec_gpu_status launch_gemm(const GemmCall& c, cudaStream_t s) {
  if (c.shape == 3) return launch_shape<MODE, T, false, 128>(c, s);
  if (c.shape == 2) return launch_shape<MODE, T, true, 128>(c, s);
  if constexpr (MODE == kLinear)
    if (c.shape == 1) return launch_shape<MODE, T, true, 192>(c, s);
  return launch_shape<MODE, T, true, 256>(c, s);
}

template <typename T>
xvec_gpu_status gemm_by_mode(const GemmCall& c, cudaStream_t s) {
  switch (c.mode) {
    case kLinear: return launch_gemm<kLinear, T>(c, s);
    case kGated: return launch_gemm<kGated, T>(c, s);
    case kDx: return launch_gemm<kDx, T>(c, s);
    default: return launch_gemm<kDw, T>(c, s);
  }
}

}  // namespace adapter
}  // namespace xvec
