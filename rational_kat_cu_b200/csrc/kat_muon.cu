// kat_muon.cu — Newton-Schulz orthogonalisation of matrix updates (C ABI: include/kat_muon.h).
//
// A call takes up to 64 matrices of one shape.  Two elementwise kernels bring the update into
// the working form (the momentum update with the sums of squares, then scaling and splitting into
// planes), then every step is three batched products on the tensor cores:
//   gram    A  = X X^T          both operands rows of X
//   poly    B  = b A + c A A    both operands rows of A (A is symmetric)
//   apply   X' = a X + B X      rows of B against X itself, read with its columns contiguous
//                               (an MN-major shared-memory operand), so X is never transposed
// gram and poly are symmetric: only the tiles on and below the diagonal are computed, and each
// is written twice, once transposed.  The last apply writes the output or updates the weights.

#include <cuda.h>  // CUtensorMap and its enums (types only: the encoder is fetched at run time)
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <mutex>

#include "kat_rational.h"
#include "kat_muon.h"

namespace {

#include "kat_math.cuh"

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;

constexpr int kMaxMats = KAT_MUON_MAX_MATRICES;
constexpr int64_t kMaxDim = 65536;
constexpr int kMaxSteps = 32;

constexpr int kTM = 128;   // output tile rows (MMA M, TMEM lanes)
constexpr int kTN = 128;   // output tile columns (MMA N, TMEM columns of one accumulator)
constexpr int kTK = 64;    // k-block: 64 fp16 = one 128-byte swizzle row
constexpr int kUmmaK = 16;
constexpr int kStages = 3;
constexpr uint32_t kPlaneBytes = kTM * kTK * 2;        // one operand plane of a stage
constexpr uint32_t kStageBytes = 4 * kPlaneBytes;      // P hi, P lo, Q hi, Q lo
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kTmemCols = 2 * kTN;
constexpr uint32_t kSmemBytes = 1024 + kStages * kStageBytes + 256;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
static_assert(kTM == kTN, "symmetric tiles are square");
constexpr long long kWaitCycles = 4000000000LL;

// Planes hold value x 2^14: the iterates' entries stay below 1.25, those of A below 1.5 and those
// of bA + cA^2 below 2.9, so 2^14 keeps the largest under fp16's 65504 and leaves the most bits
// above its subnormals.
constexpr float kScale = 16384.0f;
constexpr float kInvScale = 1.0f / 16384.0f;

__device__ int g_muon_status;

enum Mode { kGram = 0, kPoly = 1, kApply = 2, kFinal = 3 };

struct PtrTable {
  const void* p[kMaxMats];
};

// ---------------------------------------------------------------------------
// PTX wrappers.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)
               : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Bounded wait of one thread for the phase with `parity`; false when the CTA aborted or this
// wait ran out (which aborts the CTA).
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort = 1;
      atomicExch(&g_muon_status, KAT_DEVICE_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}
// The same wait without the abort flag, for teardown.
__device__ __forceinline__ void drain_phase(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (clock64() - t0 > kWaitCycles) {
      atomicExch(&g_muon_status, KAT_DEVICE_WAIT_TIMEOUT);
      return;
    }
  }
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
               : "memory");
}
// D[tmem] (+)= P[smem] Q[smem]^T for one K = 16 slice, fp16 operands.
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t p_desc, uint64_t q_desc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(p_desc), "l"(q_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar)) : "memory");
}
// 16 consecutive fp32 columns of this thread's TMEM lane, complete on return.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
        "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// Shared-memory matrix descriptors of 128-byte-swizzled tiles (start >> 4 in bits 0-13, leading
// byte offset >> 4 in 16-29, stride byte offset >> 4 in 32-45, descriptor version 1 in 46-47,
// swizzle mode 2 = 128B in 61-63).
//   K-major: rows of 64 k values; 8-row groups 1024 bytes apart; the leading offset is unused.
//   MN-major: k rows of 64 consecutive n values; 8-k groups 1024 bytes apart (stride offset),
//   blocks of 64 n one [64 k x 64 n] box apart (leading offset).
constexpr uint32_t kBoxBytes = kTK * 64 * 2;
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(kBoxBytes >> 4) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: fp32 accumulator (bits 4-5 = 1), fp16 operands (7-9, 10-12 = 0), B's
// major-ness in bit 16, N >> 3 in 17-22, M >> 4 in 24-28.
__host__ __device__ constexpr uint32_t idesc_of(bool mn_major_q) {
  return (1u << 4) | (mn_major_q ? (1u << 16) : 0u) | (uint32_t(kTN >> 3) << 17) |
         (uint32_t(kTM >> 4) << 24);
}

// ---------------------------------------------------------------------------
// Planes.
// ---------------------------------------------------------------------------

// hi + lo = v to 22 bits (v is already scaled).
__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}
__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  const __half2 h = __halves2half2(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 8 values of both planes added up.
__device__ __forceinline__ void join8(const __half* hi, const __half* lo, float (&v)[8]) {
  const uint4 h = *reinterpret_cast<const uint4*>(hi);
  const uint4 l = *reinterpret_cast<const uint4*>(lo);
  const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hw[i]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&lw[i]));
    v[2 * i] = a.x + b.x;
    v[2 * i + 1] = a.y + b.y;
  }
}

// ---------------------------------------------------------------------------
// Momentum, norm, split.
// ---------------------------------------------------------------------------

struct Update {
  PtrTable x;          // the update itself, or the gradients
  PtrTable m;          // momenta (fp32, updated), where has_momentum
  int64_t size;        // elements of a matrix
  float mu;
  int32_t nesterov;
  int32_t has_momentum;
};

template <typename T> __device__ __forceinline__ float load1(const T* p);
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float load1<__half>(const __half* p) {
  return __half2float(*p);
}
template <> __device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr int kNormThreads = 256;
constexpr int kNormBlocks = 64;  // partial sums of one matrix

// m <- mu m + g, and each block's sum of the squared update in fp64 (a gradient's square may
// leave fp32's range, and its norm is what all else is divided by).
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
kat_muon_norm_kernel(const __grid_constant__ Update u, double* __restrict__ partial) {
  const T* x = static_cast<const T*>(u.x.p[blockIdx.y]);
  float* m = static_cast<float*>(const_cast<void*>(u.m.p[blockIdx.y]));
  double sum = 0.0;
  for (int64_t i = int64_t(blockIdx.x) * kNormThreads + threadIdx.x; i < u.size;
       i += int64_t(gridDim.x) * kNormThreads) {
    float v = load1(x + i);
    if (u.has_momentum) {
      const float mom = fmaf(u.mu, m[i], v);
      m[i] = mom;
      v = u.nesterov ? fmaf(u.mu, mom, v) : mom;
    }
    sum += double(v) * double(v);
  }
  __shared__ double s[kNormThreads / 32];
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) sum += s[w];
    partial[int64_t(blockIdx.y) * kNormBlocks + blockIdx.x] = sum;
  }
}

constexpr int kSplitTile = 32;

// The scaled update in planes: X[i][j] = u / |u|_F x 2^14, rows i < m, leading dimension ld; where
// `transposed`, X = u^T.  Tiles go through shared memory so that both sides are read and written
// along their rows.
template <typename T>
__global__ void __launch_bounds__(256)
kat_muon_split_kernel(const __grid_constant__ Update u, const double* __restrict__ partial,
                      int norm_blocks, __half* __restrict__ planes, int64_t rows, int64_t cols,
                      int64_t ld, int64_t plane, int transposed, int col_tiles) {
  const int mat = blockIdx.y;
  __shared__ double s_scale;
  __shared__ float tile[kSplitTile][kSplitTile + 1];
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int b = 0; b < norm_blocks; ++b) sum += partial[int64_t(mat) * kNormBlocks + b];
    s_scale = sum > 0.0 ? double(kScale) / sqrt(sum) : (sum == 0.0 ? 0.0 : sum);
  }
  __syncthreads();
  const double scale = s_scale;
  const T* x = static_cast<const T*>(u.x.p[mat]);
  const float* m = static_cast<const float*>(u.m.p[mat]);
  const int64_t r0 = int64_t(blockIdx.x / col_tiles) * kSplitTile;
  const int64_t c0 = int64_t(blockIdx.x % col_tiles) * kSplitTile;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < kSplitTile; k += 8) {
    const int64_t r = r0 + ty + k, c = c0 + tx;
    float v = 0.0f;
    if (r < rows && c < cols) {
      const int64_t i = r * cols + c;
      v = load1(x + i);
      if (u.has_momentum) v = u.nesterov ? fmaf(u.mu, m[i], v) : m[i];
      v = float(double(v) * scale);  // the norm may lie outside fp32's range
    }
    tile[ty + k][tx] = v;
  }
  __syncthreads();
  __half* hi = planes + int64_t(mat) * 2 * plane;
  __half* lo = hi + plane;
#pragma unroll
  for (int k = 0; k < kSplitTile; k += 8) {
    int64_t i, j;
    float v;
    if (transposed) {
      i = c0 + ty + k;
      j = r0 + tx;
      v = tile[tx][ty + k];
      if (i >= cols || j >= rows) continue;
    } else {
      i = r0 + ty + k;
      j = c0 + tx;
      v = tile[ty + k][tx];
      if (i >= rows || j >= cols) continue;
    }
    __half h, l;
    split(v, h, l);
    hi[i * ld + j] = h;
    lo[i * ld + j] = l;
  }
}

// ---------------------------------------------------------------------------
// The batched product.
// ---------------------------------------------------------------------------

struct GemmArgs {
  int32_t m, n;            // output rows and columns of a matrix
  int32_t row_tiles, col_tiles, tiles;  // of one matrix; `tiles` counts the computed ones
  int32_t total_tiles;     // over all matrices
  int32_t k_blocks;
  const __half* in;        // planes the epilogue adds (poly: A, apply: X), leading dimension ld
  __half* out;             // planes written
  int64_t ld, plane;       // of both
  // final step
  int32_t transposed;
  int64_t out_ld;          // columns of the caller's matrices
  int32_t has_momentum;    // update weights instead of writing the result
  int32_t vec;             // the caller's rows take 16-byte accesses
  float lr, weight_decay, scale;
  const float* lr_device;
};

template <typename T>
__device__ __forceinline__ void final_store(const GemmArgs& args, const PtrTable& outs, int mat,
                                            int row, int col, const float (&o)[8], float lr) {
  T* base = static_cast<T*>(const_cast<void*>(outs.p[mat]));
  const float keep = 1.0f - lr * args.weight_decay, step = lr * args.scale;
  if (args.transposed) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (col + k >= args.n) break;
      T* p = base + int64_t(col + k) * args.out_ld + row;
      *p = from_float<T>(args.has_momentum ? fmaf(keep, load1(p), -step * o[k]) : o[k]);
    }
  } else if (args.vec && col + 8 <= args.n) {
    T* p = base + int64_t(row) * args.out_ld + col;
    union { uint4 q[sizeof(T) / 2]; T e[8]; } w;
    if (args.has_momentum) {
#pragma unroll
      for (int q = 0; q < int(sizeof(T) / 2); ++q) w.q[q] = reinterpret_cast<const uint4*>(p)[q];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        w.e[k] = from_float<T>(fmaf(keep, load1(&w.e[k]), -step * o[k]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w.e[k] = from_float<T>(o[k]);
    }
#pragma unroll
    for (int q = 0; q < int(sizeof(T) / 2); ++q) reinterpret_cast<uint4*>(p)[q] = w.q[q];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (col + k >= args.n) break;
      T* p = base + int64_t(row) * args.out_ld + col + k;
      *p = from_float<T>(args.has_momentum ? fmaf(keep, load1(p), -step * o[k]) : o[k]);
    }
  }
}

template <int kMode, typename T>
__global__ void __launch_bounds__(kThreads, 1)
kat_muon_gemm_kernel(const __grid_constant__ CUtensorMap tm_p,
                     const __grid_constant__ CUtensorMap tm_q,
                     const __grid_constant__ GemmArgs args,
                     const __grid_constant__ PtrTable outs) {
  constexpr bool kSym = kMode == kGram || kMode == kPoly;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int j = 0; j < 2; ++j) {
      mbar_init(tfull + j, 1);
      mbar_init(tempty + j, kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tm_p);
    prefetch_map(&tm_q);
  }
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Tile -> matrix, row tile, column tile (row >= column where the product is symmetric).
  auto locate = [&](int tile, int& mat, int& tr, int& tc) {
    mat = tile / args.tiles;
    const int t = tile - mat * args.tiles;
    if (kSym) {
      tr = int((sqrtf(8.0f * float(t) + 1.0f) - 1.0f) * 0.5f);
      while ((tr + 1) * (tr + 2) / 2 <= t) ++tr;
      while (tr * (tr + 1) / 2 > t) --tr;
      tc = t - tr * (tr + 1) / 2;
    } else {
      tr = t % args.row_tiles;
      tc = t / args.row_tiles;
    }
  };

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, wrapped = false;
      for (int tile = blockIdx.x; tile < args.total_tiles && ok; tile += gridDim.x) {
        int mat, tr, tc;
        locate(tile, mat, tr, tc);
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!wait_phase(empty + stage, phase ^ 1u, abort)) { ok = false; break; }
          uint8_t* s = smem + stage * kStageBytes;
          mbar_expect_tx(full + stage, kStageBytes);
          for (int h = 0; h < 2; ++h) {
            tma_load_3d(s + h * kPlaneBytes, &tm_p, full + stage, kb * kTK, tr * kTM,
                        2 * mat + h);
            uint8_t* q = s + (2 + h) * kPlaneBytes;
            if (kSym) {
              tma_load_3d(q, &tm_q, full + stage, kb * kTK, tc * kTN, 2 * mat + h);
            } else {
              tma_load_3d(q, &tm_q, full + stage, tc * kTN, kb * kTK, 2 * mat + h);
              tma_load_3d(q + kBoxBytes, &tm_q, full + stage, tc * kTN + 64, kb * kTK,
                          2 * mat + h);
            }
          }
          if (++stage == kStages) { stage = 0; phase ^= 1u; wrapped = true; }
        }
      }
      if (!ok) {
        // given up: the copies in flight land before the block ends
        for (int s = 0; s < kStages; ++s)
          if (s < stage || wrapped) drain_phase(full + s, s < stage ? phase : phase ^ 1u);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool issued = false, ok = true;
      for (int tile = blockIdx.x; tile < args.total_tiles && ok; tile += gridDim.x, ++local) {
        const int acc = local & 1;
        if (!wait_phase(tempty + acc, ((local >> 1) & 1) ^ 1u, abort)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + uint32_t(acc * kTN);
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!wait_phase(full + stage, phase, abort)) { ok = false; break; }
          tc_fence_after();
          const uint32_t s = smem_u32(smem + stage * kStageBytes);
          const uint64_t p_hi = desc_k(s), p_lo = desc_k(s + kPlaneBytes);
          const uint64_t q_hi = kSym ? desc_k(s + 2 * kPlaneBytes) : desc_mn(s + 2 * kPlaneBytes);
          const uint64_t q_lo = kSym ? desc_k(s + 3 * kPlaneBytes) : desc_mn(s + 3 * kPlaneBytes);
          // a K = 16 slice further: 32 bytes inside the swizzled rows (K-major), two 8-k groups
          // (MN-major)
          constexpr uint64_t kStepP = 32 >> 4, kStepQ = kSym ? (32 >> 4) : (2048 >> 4);
          constexpr uint32_t idesc = idesc_of(!kSym);
#pragma unroll
          for (int k = 0; k < kTK / kUmmaK; ++k) {
            umma_f16(d, p_hi + k * kStepP, q_hi + k * kStepQ, idesc, (kb | k) != 0 ? 1u : 0u);
            umma_f16(d, p_hi + k * kStepP, q_lo + k * kStepQ, idesc, 1u);
            umma_f16(d, p_lo + k * kStepP, q_hi + k * kStepQ, idesc, 1u);
          }
          issued = true;
          umma_commit(empty + stage);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok) umma_commit(tfull + acc);
      }
      if (issued) {
        // Every MMA has completed before the tensor memory is freed.
        umma_commit(drain);
        drain_phase(drain, 0);
      }
    }
  } else {
    // ---------------- epilogue: a TMEM lane quadrant and a column half per warp ----------------
    const int ew = warp - 2;
    const int quad = warp & 3;
    const int half = ew >> 2;
    const uint32_t lane_addr = tmem_base + (uint32_t(quad * 32) << 16);
    const float lr = kMode == kFinal && args.has_momentum && args.lr_device != nullptr
                         ? *args.lr_device : args.lr;
    int local = 0;
    for (int tile = blockIdx.x; tile < args.total_tiles; tile += gridDim.x, ++local) {
      const int acc = local & 1;
      int mat, tr, tc;
      locate(tile, mat, tr, tc);
      int ok = 1;
      if (lane == 0) ok = wait_phase(tfull + acc, (local >> 1) & 1, abort) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      (void)mbar_try(tfull + acc, (local >> 1) & 1);  // completed: acquire for every lane
      tc_fence_after();
      const int row = tr * kTM + quad * 32 + lane;
      const __half* in_hi = args.in + int64_t(mat) * 2 * args.plane;
      __half* out_hi = args.out + int64_t(mat) * 2 * args.plane;
      for (int c = 0; c < 4; ++c) {
        const int col0 = tc * kTN + half * 64 + c * 16;
        uint32_t v[16];
        tmem_ld16(lane_addr + uint32_t(acc * kTN + half * 64 + c * 16), v);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int col = col0 + g * 8;
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = __uint_as_float(v[g * 8 + k]) * kInvScale;
          const bool inside = row < args.m && col < int(args.ld);  // ld is a multiple of 8
          if (kMode != kGram && inside) {
            float x[8];
            const int64_t at = int64_t(row) * args.ld + col;
            join8(in_hi + at, in_hi + args.plane + at, x);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              y[k] = kMode == kPoly ? fmaf(kB, x[k], kC * y[k]) : fmaf(kA, x[k], y[k]);
          }
          if constexpr (kMode == kFinal) {
            if (inside && col < args.n) {
#pragma unroll
              for (int k = 0; k < 8; ++k) y[k] *= kInvScale;
              final_store<T>(args, outs, mat, row, col, y, lr);
            }
          } else {
            __half hi[8], lo[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) split(y[k], hi[k], lo[k]);
            if (inside) {
              const int64_t at = int64_t(row) * args.ld + col;
              *reinterpret_cast<uint4*>(out_hi + at) =
                  make_uint4(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]), pack2(hi[4], hi[5]),
                             pack2(hi[6], hi[7]));
              *reinterpret_cast<uint4*>(out_hi + args.plane + at) =
                  make_uint4(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(lo[4], lo[5]),
                             pack2(lo[6], lo[7]));
            }
            if (kSym && tr != tc && row < args.m) {
              // the mirror image: for one column the warp's 32 rows are consecutive
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if (col + k < args.n) {
                  const int64_t at = int64_t(col + k) * args.ld + row;
                  out_hi[at] = hi[k];
                  out_hi[args.plane + at] = lo[k];
                }
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty + acc);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Planes [2 x count][rows][ld] of which `cols` columns count: what lies beyond rows or cols is
// read as zero, so no tile edge needs padding in memory.
bool make_map(CUtensorMap* map, const __half* base, int64_t planes, int64_t rows, int64_t cols,
              int64_t ld, uint32_t box_rows) {
  EncodeTiledFn fn = encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * cuuint64_t(rows) * 2};
  const cuuint32_t box[3] = {64, box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count(int device) {
  static std::mutex mu;
  static int cache[64] = {0};
  std::lock_guard<std::mutex> lock(mu);
  if (device < 0 || device >= 64) return 0;
  if (cache[device] == 0) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
      return 0;
    cache[device] = v;
  }
  return cache[device];
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Where each part of the workspace lies (bytes; every part a multiple of 256).
struct Layout {
  int64_t m, n, ldn, ldm, plane_x, plane_a;
  size_t x0, x1, a, b, partial, total;
  Layout(int64_t count, int64_t rows, int64_t cols) {
    m = rows < cols ? rows : cols;
    n = rows < cols ? cols : rows;
    ldn = round_up(n, 8);
    ldm = round_up(m, 8);
    plane_x = m * ldn;
    plane_a = m * ldm;
    const size_t bx = size_t(round_up(count * 2 * plane_x * 2, 256));
    const size_t ba = size_t(round_up(count * 2 * plane_a * 2, 256));
    x0 = 0;
    x1 = x0 + bx;
    a = x1 + bx;
    b = a + ba;
    partial = b + ba;
    total = partial + size_t(round_up(count * kNormBlocks * int64_t(sizeof(double)), 256));
  }
};

int check_args(int32_t count, int64_t rows, int64_t cols, int32_t dtype, int32_t steps) {
  if (dtype != KAT_DTYPE_F32 && dtype != KAT_DTYPE_F16 && dtype != KAT_DTYPE_BF16)
    return KAT_ERR_BAD_DTYPE;
  if (count < 0 || count > kMaxMats || rows < 1 || cols < 1 || rows > kMaxDim || cols > kMaxDim ||
      steps < 1 || steps > kMaxSteps)
    return KAT_ERR_BAD_SHAPE;
  return KAT_OK;
}

template <int kMode, typename T>
int launch_gemm(const CUtensorMap& p, const CUtensorMap& q, const GemmArgs& args,
                const PtrTable& outs, int sms, cudaStream_t stream) {
  auto kernel = kat_muon_gemm_kernel<kMode, T>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(kSmemBytes)) != cudaSuccess)
    return KAT_ERR_CUDA;
  const int grid = args.total_tiles < sms ? args.total_tiles : sms;
  kernel<<<grid, kThreads, kSmemBytes, stream>>>(p, q, args, outs);
  return cudaGetLastError() == cudaSuccess ? KAT_OK : KAT_ERR_CUDA;
}

template <typename T>
int run(const Update& u, const PtrTable& outs, GemmArgs fin, int32_t count, int64_t rows,
        int64_t cols, int32_t steps, uint8_t* ws, int sms, cudaStream_t stream) {
  const Layout L(count, rows, cols);
  __half* x[2] = {reinterpret_cast<__half*>(ws + L.x0), reinterpret_cast<__half*>(ws + L.x1)};
  __half* a = reinterpret_cast<__half*>(ws + L.a);
  __half* b = reinterpret_cast<__half*>(ws + L.b);
  double* partial = reinterpret_cast<double*>(ws + L.partial);
  const int transposed = rows > cols;

  int64_t want = (u.size + kNormThreads * 16 - 1) / (kNormThreads * 16);
  const int norm_blocks = int(want < kNormBlocks ? want : kNormBlocks);
  kat_muon_norm_kernel<T><<<dim3(norm_blocks, count), kNormThreads, 0, stream>>>(u, partial);
  const int row_tiles = int((rows + kSplitTile - 1) / kSplitTile);
  const int col_tiles = int((cols + kSplitTile - 1) / kSplitTile);
  kat_muon_split_kernel<T><<<dim3(uint32_t(row_tiles) * col_tiles, count), 256, 0, stream>>>(
      u, partial, norm_blocks, x[0], rows, cols, L.ldn, L.plane_x, transposed, col_tiles);
  if (cudaGetLastError() != cudaSuccess) return KAT_ERR_CUDA;

  CUtensorMap xk[2], xmn[2], ma, mb;
  for (int i = 0; i < 2; ++i)
    if (!make_map(&xk[i], x[i], 2 * count, L.m, L.n, L.ldn, kTM) ||
        !make_map(&xmn[i], x[i], 2 * count, L.m, L.n, L.ldn, kTK))
      return KAT_ERR_CUDA;
  if (!make_map(&ma, a, 2 * count, L.m, L.m, L.ldm, kTM) ||
      !make_map(&mb, b, 2 * count, L.m, L.m, L.ldm, kTM))
    return KAT_ERR_CUDA;

  const int tm = int((L.m + kTM - 1) / kTM), tn = int((L.n + kTN - 1) / kTN);
  GemmArgs sym{};
  sym.m = sym.n = int32_t(L.m);
  sym.row_tiles = sym.col_tiles = tm;
  sym.tiles = tm * (tm + 1) / 2;
  sym.total_tiles = sym.tiles * count;
  sym.ld = L.ldm;
  sym.plane = L.plane_a;
  fin.m = int32_t(L.m);
  fin.n = int32_t(L.n);
  fin.row_tiles = tm;
  fin.col_tiles = tn;
  fin.tiles = tm * tn;
  fin.total_tiles = fin.tiles * count;
  fin.k_blocks = int((L.m + kTK - 1) / kTK);
  fin.ld = L.ldn;
  fin.plane = L.plane_x;
  fin.transposed = transposed;
  fin.out_ld = cols;
  for (int s = 0; s < steps; ++s) {
    const int cur = s & 1;
    GemmArgs g = sym;
    g.k_blocks = int((L.n + kTK - 1) / kTK);
    g.in = g.out = a;
    if (int rc = launch_gemm<kGram, float>(xk[cur], xk[cur], g, outs, sms, stream)) return rc;
    g.k_blocks = fin.k_blocks;
    g.in = a;
    g.out = b;
    if (int rc = launch_gemm<kPoly, float>(ma, ma, g, outs, sms, stream)) return rc;
    fin.in = x[cur];
    fin.out = x[cur ^ 1];
    const int rc = s + 1 < steps
                       ? launch_gemm<kApply, float>(mb, xmn[cur], fin, outs, sms, stream)
                       : launch_gemm<kFinal, T>(mb, xmn[cur], fin, outs, sms, stream);
    if (rc) return rc;
  }
  return KAT_OK;
}

int dispatch(const Update& u, const PtrTable& outs, const GemmArgs& fin, int32_t count,
             int64_t rows, int64_t cols, int32_t dtype, int32_t steps, void* ws, size_t ws_bytes,
             void* stream) {
  const Layout L(count, rows, cols);
  if (ws == nullptr || ws_bytes < L.total || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
    return KAT_ERR_WORKSPACE;
  // tiles of all matrices are counted in 32 bits
  const int64_t tm = (L.m + kTM - 1) / kTM, tn = (L.n + kTN - 1) / kTN;
  if (tm * tn * count >= (int64_t(1) << 30)) return KAT_ERR_BAD_SHAPE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KAT_ERR_CUDA;
  const int sms = sm_count(dev);
  if (sms <= 0) return KAT_ERR_CUDA;
  uint8_t* w = static_cast<uint8_t*>(ws);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KAT_DTYPE_F32: return run<float>(u, outs, fin, count, rows, cols, steps, w, sms, st);
    case KAT_DTYPE_F16: return run<__half>(u, outs, fin, count, rows, cols, steps, w, sms, st);
    default: return run<__nv_bfloat16>(u, outs, fin, count, rows, cols, steps, w, sms, st);
  }
}

}  // namespace

extern "C" {

size_t kat_muon_workspace_bytes(int32_t count, int64_t rows, int64_t cols) {
  if (check_args(count, rows, cols, KAT_DTYPE_F32, 1) != KAT_OK || count == 0) return 0;
  return Layout(count, rows, cols).total;
}

int kat_orthogonalize(const void* const* x, void* const* out, int32_t count, int64_t rows,
                      int64_t cols, int32_t dtype, int32_t steps, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (int st = check_args(count, rows, cols, dtype, steps)) return st;
  if (count == 0) return KAT_OK;
  if (x == nullptr || out == nullptr) return KAT_ERR_NULL_POINTER;
  Update u{};
  PtrTable outs{};
  GemmArgs fin{};
  u.size = rows * cols;
  fin.vec = cols % 8 == 0;
  for (int i = 0; i < count; ++i) {
    if (x[i] == nullptr || out[i] == nullptr) return KAT_ERR_NULL_POINTER;
    u.x.p[i] = x[i];
    outs.p[i] = out[i];
    if ((reinterpret_cast<uintptr_t>(out[i]) & 15u) != 0) fin.vec = 0;
  }
  return dispatch(u, outs, fin, count, rows, cols, dtype, steps, workspace, workspace_bytes,
                  stream);
}

int kat_muon_step(void* const* weights, const void* const* grads, float* const* momenta,
                  int32_t count, int64_t rows, int64_t cols, int32_t dtype, float lr,
                  const float* lr_device, float momentum, int32_t nesterov, float weight_decay,
                  float scale, int32_t steps, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (int st = check_args(count, rows, cols, dtype, steps)) return st;
  if (count == 0) return KAT_OK;
  if (weights == nullptr || grads == nullptr || momenta == nullptr) return KAT_ERR_NULL_POINTER;
  Update u{};
  PtrTable outs{};
  GemmArgs fin{};
  u.size = rows * cols;
  u.mu = momentum;
  u.nesterov = nesterov != 0;
  u.has_momentum = 1;
  fin.has_momentum = 1;
  fin.lr = lr;
  fin.lr_device = lr_device;
  fin.weight_decay = weight_decay;
  fin.scale = scale;
  fin.vec = cols % 8 == 0;
  for (int i = 0; i < count; ++i) {
    if (weights[i] == nullptr || grads[i] == nullptr || momenta[i] == nullptr)
      return KAT_ERR_NULL_POINTER;
    u.x.p[i] = grads[i];
    u.m.p[i] = momenta[i];
    outs.p[i] = weights[i];
    if ((reinterpret_cast<uintptr_t>(weights[i]) & 15u) != 0) fin.vec = 0;
  }
  return dispatch(u, outs, fin, count, rows, cols, dtype, steps, workspace, workspace_bytes,
                  stream);
}

int kat_muon_device_status(int device, int reset, int* status) {
  if (status == nullptr) return KAT_ERR_NULL_POINTER;
  int prev = 0;
  if (cudaGetDevice(&prev) != cudaSuccess) return KAT_ERR_CUDA;
  if (device != prev && cudaSetDevice(device) != cudaSuccess) return KAT_ERR_CUDA;
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_muon_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_muon_status, &zero, sizeof(int));
  }
  if (device != prev) cudaSetDevice(prev);
  if (e != cudaSuccess) return KAT_ERR_CUDA;
  *status = v;
  return KAT_OK;
}

}  // extern "C"
