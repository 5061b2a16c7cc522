// kat_muon.cu — Newton-Schulz orthogonalisation of matrix updates (C ABI: include/kat_muon.h).
//
// A call takes up to 64 matrices of one shape, m <= n.  Two elementwise kernels bring the update into
// the working form (the momentum update with the sums of squares, then scaling and splitting into
// planes); all else is batched products on the tensor cores.  One step of the iteration is
//   gram    A  = X X^T                  both operands rows of X
//   poly    P  = a I + b A + c A A      both operands rows of A (A is symmetric)
//   apply   X' = P X                    rows of P against X itself, read with its columns contiguous
//                                       (an MN-major shared-memory operand): X is never transposed
// gram, poly and all other m x m products are symmetric: only the tiles on and below the diagonal
// are computed and stored.  Where a product needs a block above it, it reads the block below with
// its columns contiguous, the same way as X: each k-block's instruction descriptor says which way
// its operands lie.  (Writing each tile a second time, transposed, took as long as the MMAs.)  The
// last apply writes the output or updates the weights.
//
// Wide matrices take up to three steps at once on the Gram matrix: the next step's is
// A' = P A P (all of these commute), and X is multiplied once by the product of the P's:
// 6 m^2 n + 14 m^3 operations for five steps in blocks of 3 and 2, instead of 15 m^2 n + 5 m^3
// (products of two factors counted by halves).  Taking all five steps at once would cost
// 3 m^2 n + 17 m^3 but loses digits where the singular values spread (relative error 2.7e-4 against
// 1.4e-5 of fp32 products for singular values 1 / k; blocks of 3 and 2: 1.3e-5).
//
// Up to 128 rows one CTA takes a block's whole chain of m x m products, from A to the product of the
// P's, in its shared memory: a product of that size is over in 2 us, half the time of a launch.
// (Clusters that share a tile's K blocks and hand each other partial sums did not pay: the sums'
// way through distributed shared memory took 7000 cycles, as long as the MMAs it saved.)
//
// Each product of two split matrices takes three MMAs (hi hi, hi lo, lo hi) on four operand planes.
// With one CTA to a 128 x 128 tile the planes' way from L2 is what bounds it (64 KB a k-block for
// 768 cycles of MMA); a CTA pair (cta_group::2) on a 256 x 256 tile loads the same bytes for twice
// the MMAs.  Launches overlap by programmatic dependent launch: a kernel sets up its barriers and
// tensor memory while the one before it ends.

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

constexpr int kTM = 128;   // operand rows of a CTA: its tile rows, and its share of the columns
constexpr int kTK = 64;    // k-block: 64 fp16 = one 128-byte swizzle row
constexpr int kUmmaK = 16;
constexpr uint32_t kPlaneBytes = kTM * kTK * 2;        // one operand plane of a stage
constexpr uint32_t kRingBytes = 12 * kPlaneBytes;      // stages: 3 of P and Q in two planes
constexpr int kMaxStages = 4;                          // (half tiles: 4)
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kPiece = 32;         // rows and columns an epilogue warp handles at once
constexpr uint32_t kStagingBytes = 2 * kPiece * kPiece * 2;   // of a warp: a piece in two planes
constexpr uint32_t kSmemBytes = 1024 + kRingBytes + kEpiWarps * kStagingBytes + 256;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
constexpr long long kWaitCycles = 4000000000LL;

// Planes of X, A and P hold value x 2^14: the iterates' entries stay below 1.25, those of A below 1.5
// and those of P below 3.45, so 2^14 keeps the largest under fp16's 65504 and leaves the most bits
// above its subnormals.  A product of k P's reaches 3.45^k and holds value x 2^(16 - 2k).
constexpr float kScale = 16384.0f;
constexpr int kMaxBlock = 3;   // steps taken on the Gram matrix at once

// k-blocks that one accumulator takes at most.  The tensor cores cut what they add, so a sum loses the
// more the longer it is (always the same way where its terms have one sign, as on A's diagonal):
// undivided, five steps of [128,65536] were off by 1e-3, three of [256,65536] by 3.3e-4 and five of
// [4096,4096] by 1.0e-4; in parts of 16 by 2.2e-5, 4.2e-6 and 2.8e-5.  The parts are added up in fp32, with
// rounding, while the MMAs wait for their accumulator: nothing up to 1024 terms, 1 % of
// 12 x [768,2304], 4 % of [4096,4096].  (Parts of 8: half the error from 768 terms on, 3 to 6 %
// slower everywhere.)
constexpr int kSumBlocks = 16;

__device__ int g_muon_status;

enum Mode { kGram = 0, kSym = 1, kPoly = 2, kApply = 3, kFinal = 4 };

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
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int32_t x,
                                             int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_read() {   // earlier stores have read their source
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
template <int kPair>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  if constexpr (kPair == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int kPair>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  if constexpr (kPair == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
                 : "memory");
  } else {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
                 : "memory");
  }
}
// D[tmem] (+)= P[smem] Q[smem]^T for one K = 16 slice, fp16 operands.  The whole warp comes here with
// the same operands, and its `leader` lane issues.
template <int kPair>
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t p_desc, uint64_t q_desc,
                                         uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  if constexpr (kPair == 1) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(p_desc), "l"(q_desc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(p_desc), "l"(q_desc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
  }
}
// One lane of a whole warp.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t mine;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(mine));
  return mine;
}
// Arrive on the mbarrier at shared::cluster address `bar` when every MMA this thread issued so far
// has completed.
template <int kPair>
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  if constexpr (kPair == 1) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     bar) : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     bar) : "memory");
  }
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" :::
                   "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}
// Load into this CTA's shared memory whose completion is counted on the pair's rank-0 barrier.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// Programmatic dependent launch: let the next kernel's blocks start; wait until the kernel before
// has completed and its writes are visible.
__device__ __forceinline__ void pdl_launch_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// 16 values into consecutive columns of this thread's TMEM lane (complete after tmem_st_wait).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
      "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
      "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])), "r"(__float_as_uint(v[8])),
      "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])),
      "r"(__float_as_uint(v[15]))
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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
// Instruction descriptor: fp32 accumulator (bits 4-5 = 1), fp16 operands (7-9, 10-12 = 0), the
// operands' major-ness in bits 15 and 16 (1: MN-major), N >> 3 in 17-22, M >> 4 in 24-28; tiles are
// 128 rows by kCols columns or (a CTA pair) 256 square.
template <int kPair, int kCols>
__host__ __device__ constexpr uint32_t idesc_of(bool mn_p, bool mn_q) {
  return (1u << 4) | (mn_p ? (1u << 15) : 0u) | (mn_q ? (1u << 16) : 0u) |
         (uint32_t((kCols * kPair) >> 3) << 17) | (uint32_t((kTM * kPair) >> 4) << 24);
}

template <auto V> struct Const { static constexpr auto value = V; };

// The MMAs of one k-block: operands at shared addresses p and q, their second planes `step_p` and
// `step_q` further, accumulator d.  Which way the operands lie is a template parameter: with descriptors that
// depend on run-time values each MMA took 270 cycles to issue, four times its execution.  And the whole
// warp comes here: in a branch of one lane each took 83 cycles, now 65 at most (one [768,768] bf16: 168
// -> 145 us).
template <int kPair, int kCols, bool kMnP, bool kMnQ>
__device__ __forceinline__ void issue_block(uint32_t d, uint32_t p, uint32_t q, uint32_t step_p,
                                            uint32_t step_q, bool accumulate, uint32_t leader) {
  const uint64_t p_hi = kMnP ? desc_mn(p) : desc_k(p), q_hi = kMnQ ? desc_mn(q) : desc_k(q);
  const uint64_t p_lo = kMnP ? desc_mn(p + step_p) : desc_k(p + step_p);
  const uint64_t q_lo = kMnQ ? desc_mn(q + step_q) : desc_k(q + step_q);
  // a K = 16 slice further: 32 bytes inside the swizzled rows (K-major), two 8-k groups (MN-major)
  constexpr uint64_t kStepP = kMnP ? (2048 >> 4) : (32 >> 4), kStepQ = kMnQ ? (2048 >> 4) : (32 >> 4);
  constexpr uint32_t idesc = idesc_of<kPair, kCols>(kMnP, kMnQ);
#pragma unroll
  for (int k = 0; k < kTK / kUmmaK; ++k) {
    umma_f16<kPair>(d, p_hi + k * kStepP, q_hi + k * kStepQ, idesc, accumulate || k != 0 ? 1u : 0u,
                    leader);
    umma_f16<kPair>(d, p_hi + k * kStepP, q_lo + k * kStepQ, idesc, 1u, leader);
    umma_f16<kPair>(d, p_lo + k * kStepP, q_hi + k * kStepQ, idesc, 1u, leader);
  }
}

// ---------------------------------------------------------------------------
// Planes.
// ---------------------------------------------------------------------------

// 8 scaled values in planes: hi + lo = v to 22 bits.  Two values to a conversion: one at a time they
// took most of an epilogue.
__device__ __forceinline__ void split8(const float* v, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    h[i] = *reinterpret_cast<const uint32_t*>(&a);
    l[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// 8 values of both planes added up.
__device__ __forceinline__ void join8(const uint4& h, const uint4& l, float (&v)[8]) {
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

// V neighbouring values as fp32: 8 at once where the matrices start on 16 bytes, else one.
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = load1(p);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 v = reinterpret_cast<const float4*>(p)[q];
      f[4 * q] = v.x; f[4 * q + 1] = v.y; f[4 * q + 2] = v.z; f[4 * q + 3] = v.w;
    }
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 h = Codec<T>::unpack_word(w[q]);
      f[2 * q] = h.x;
      f[2 * q + 1] = h.y;
    }
  }
}

// The update at element i, momentum already renewed.
template <typename T, int V>
__device__ __forceinline__ void load_update(const Update& u, const T* x, const float* m, int64_t i,
                                            float (&f)[V]) {
  load_values<T, V>(x + i, f);
  if (u.has_momentum) {
    float mom[V];
    load_values<float, V>(m + i, mom);
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = u.nesterov ? fmaf(u.mu, mom[k], f[k]) : mom[k];
  }
}

// m <- mu m + g, and each block's sum of the squared update in fp64 (a gradient's square may
// leave fp32's range, and its norm is what all else is divided by).
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads)
kat_muon_norm_kernel(const __grid_constant__ Update u, double* __restrict__ partial) {
  pdl_launch_next();
  const T* x = static_cast<const T*>(u.x.p[blockIdx.y]);
  float* m = static_cast<float*>(const_cast<void*>(u.m.p[blockIdx.y]));
  double sum = 0.0;
#pragma unroll 2
  for (int64_t i = (int64_t(blockIdx.x) * kNormThreads + threadIdx.x) * V; i < u.size;
       i += int64_t(gridDim.x) * kNormThreads * V) {
    float f[V];
    load_values<T, V>(x + i, f);
    if (u.has_momentum) {
      float mom[V];
      load_values<float, V>(m + i, mom);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        mom[k] = fmaf(u.mu, mom[k], f[k]);
        f[k] = u.nesterov ? fmaf(u.mu, mom[k], f[k]) : mom[k];
      }
      if constexpr (V == 1) {
        m[i] = mom[0];
      } else {
#pragma unroll
        for (int q = 0; q < V / 4; ++q)
          reinterpret_cast<float4*>(m + i)[q] =
              make_float4(mom[4 * q], mom[4 * q + 1], mom[4 * q + 2], mom[4 * q + 3]);
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) sum += double(f[k]) * double(f[k]);
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

// 2^14 / |u|_F of a matrix, by one warp: 0 for a zero update, NaN where the sum is.
__device__ __forceinline__ double scale_of(const double* partial, int blocks) {
  const int lane = threadIdx.x & 31;
  double sum = (lane < blocks ? partial[lane] : 0.0) + (lane + 32 < blocks ? partial[lane + 32] : 0.0);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  return sum > 0.0 ? double(kScale) / sqrt(sum) : (sum == 0.0 ? 0.0 : sum);
}
static_assert(kNormBlocks == 64, "scale_of adds two partial sums a lane");

constexpr int kSplitTile = 64;
constexpr int kSplitThreads = 256;

// The scaled update in planes: X[i][j] = u / |u|_F x 2^14, rows i < m, leading dimension ld; where
// `transposed`, X = u^T.  64 x 64 tiles go through shared memory, so that both sides are read and
// written along their rows, 8 values a thread.
template <typename T, int V>
__global__ void __launch_bounds__(kSplitThreads)
kat_muon_split_kernel(const __grid_constant__ Update u, const double* __restrict__ partial,
                      int norm_blocks, __half* __restrict__ planes, int64_t rows, int64_t cols,
                      int64_t ld, int64_t plane, int transposed, int col_tiles) {
  pdl_launch_next();
  pdl_wait_previous();
  const int mat = blockIdx.y;
  __shared__ double s_scale;
  __shared__ float tile[kSplitTile][kSplitTile + 1];
  if (threadIdx.x < 32) {
    const double v = scale_of(partial + int64_t(mat) * kNormBlocks, norm_blocks);
    if (threadIdx.x == 0) s_scale = v;
  }
  const T* x = static_cast<const T*>(u.x.p[mat]);
  const float* m = static_cast<const float*>(u.m.p[mat]);
  const int64_t r0 = int64_t(blockIdx.x / col_tiles) * kSplitTile;
  const int64_t c0 = int64_t(blockIdx.x % col_tiles) * kSplitTile;
  constexpr int kAcross = kSplitTile / V;                 // pieces of a tile's row
  constexpr int kPasses = kSplitTile * kAcross / kSplitThreads;
  const int px = threadIdx.x % kAcross, py = threadIdx.x / kAcross;
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int tr = py + k * (kSplitThreads / kAcross);
    const int64_t r = r0 + tr, c = c0 + px * V;
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = 0.0f;
    if (r < rows && c < cols) load_update<T, V>(u, x, m, r * cols + c, f);  // cols % V == 0
#pragma unroll
    for (int e = 0; e < V; ++e) tile[tr][px * V + e] = f[e];
  }
  __syncthreads();
  const double scale = s_scale;
  __half* hi = planes + int64_t(mat) * 2 * plane;
  __half* lo = hi + plane;
  const int64_t i0 = transposed ? c0 : r0, j0 = transposed ? r0 : c0;
  const int64_t height = transposed ? cols : rows;
#pragma unroll
  for (int k = 0; k < kSplitTile * kSplitTile / 8 / kSplitThreads; ++k) {
    const int piece = threadIdx.x + k * kSplitThreads;
    const int ti = piece / 8, tj = piece % 8 * 8;
    const int64_t i = i0 + ti, j = j0 + tj;
    if (i >= height || j >= ld) continue;                // ld is a multiple of 8
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = transposed ? tile[tj + e][ti] : tile[ti][tj + e];
      v[e] = float(double(f) * scale);                   // the norm may lie outside fp32's range
    }
    uint4 h, l;
    split8(v, h, l);
    *reinterpret_cast<uint4*>(hi + i * ld + j) = h;
    *reinterpret_cast<uint4*>(lo + i * ld + j) = l;
  }
}

// ---------------------------------------------------------------------------
// The batched product.
// ---------------------------------------------------------------------------

struct GemmArgs {
  int32_t m, n;            // output rows and columns of a matrix
  int32_t row_tiles;
  int32_t tiles;           // computed tiles of one matrix
  int32_t set_tiles;       // of all matrices of one set of operands
  int32_t total_tiles;     // of both sets
  int32_t k_blocks;
  int32_t part_blocks;     // k-blocks of an accumulator (the last one's may be fewer)
  float mult[2];           // accumulator -> plane (or, last, output) value, by set
  const __half* in;        // poly: planes of A
  int64_t ld, plane;
  // final step
  int32_t transposed;
  int64_t out_ld;          // columns of the caller's matrices
  int32_t has_momentum;    // update weights instead of writing the result
  float lr, weight_decay, scale;
  const float* lr_device;
};

// 32 fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void read_piece(uint32_t taddr, float (&y)[kPiece]) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    uint32_t v[16];
    tmem_ld16(taddr + uint32_t(g * 16), v);
#pragma unroll
    for (int k = 0; k < 16; ++k) y[g * 16 + k] = __uint_as_float(v[k]);
  }
}

// 32 columns at `from` added to those at `to`.
__device__ __forceinline__ void add_piece(uint32_t to, uint32_t from) {
  float y[kPiece], x[kPiece];
  read_piece(from, y);
  read_piece(to, x);
#pragma unroll
  for (int k = 0; k < kPiece; ++k) x[k] += y[k];
  tmem_st16(to, x);
  tmem_st16(to + 16, x + 16);
}

// Staging of a warp.  Planes: 32 rows of 64 bytes, 16-byte granules swizzled as TMA's 64-byte mode
// has it (granule index XOR address bits 7-8), so that neither rows nor granules collide.
__device__ __forceinline__ uint32_t plane_offset(int row, int granule) {
  return uint32_t(row) * 64u + uint32_t((granule ^ ((row >> 1) & 3)) << 4);
}

// kCols: columns of the output that a CTA's rows of Q make, 128, or 64 (half tiles, single CTAs only).
template <int kMode, typename T, int kPair, int kCols>
__global__ void __launch_bounds__(kThreads, 1)
kat_muon_gemm_kernel(const __grid_constant__ CUtensorMap tm_p,
                     const __grid_constant__ CUtensorMap tm_q0,
                     const __grid_constant__ CUtensorMap tm_q1,
                     const __grid_constant__ CUtensorMap tm_out0,
                     const __grid_constant__ CUtensorMap tm_out1,
                     const __grid_constant__ GemmArgs args,
                     const __grid_constant__ PtrTable outs) {
  constexpr bool kLower = kMode == kGram || kMode == kSym || kMode == kPoly;  // symmetric output
  constexpr bool kSymP = kMode != kGram, kSymQ = kMode == kSym || kMode == kPoly;
  constexpr bool kColsQ = kMode == kApply || kMode == kFinal;   // Q is X, by its columns
  constexpr int kTile = kTM * kPair;                  // output tile, square
  constexpr int kParts = kTM / kCols;                 // of its columns, each a tile of its own here
  constexpr int kAccCols = kCols * kPair;
  constexpr uint32_t kTmemCols = 2 * kAccCols;        // two accumulators
  constexpr uint32_t kQBytes = kPlaneBytes / kParts;  // an operand plane of Q in a stage
  static_assert(kParts == 1 || kPair == 1, "pairs take whole tiles");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = smem + kRingBytes;   // [epilogue warp]
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kEpiWarps * kStagingBytes);
  uint64_t* empty = full + kMaxStages;   // in each CTA
  uint64_t* tfull = empty + kMaxStages;  // in each CTA
  uint64_t* tempty = tfull + 2;       // rank 0's counts the epilogue warps of both CTAs
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_launch_next();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair == 2 ? cluster_rank() : 0u;
  const int slot0 = int(blockIdx.x) / kPair, slots = int(gridDim.x) / kPair;

  constexpr int stages = kParts == 1 ? 3 : 4;
  constexpr uint32_t stage_bytes = 2 * (kPlaneBytes + kQBytes);
  static_assert(stages <= kMaxStages && stages * stage_bytes <= kRingBytes, "ring");
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int j = 0; j < 2; ++j) {
      mbar_init(tfull + j, 1);
      mbar_init(tempty + j, kPair * kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tm_p);
    prefetch_map(&tm_q0);
    if (kMode != kFinal) prefetch_map(&tm_out0);
  }
  if (warp == 1) tmem_alloc<kPair>(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair == 2) cluster_sync();  // the peer's barriers exist before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait_previous();

  // Tile -> set, matrix, row tile, column tile (row >= column where the product is symmetric) and
  // the first column in it.
  auto locate = [&](int tile, int& set, int& mat, int& tr, int& tc, int& part) {
    part = tile % kParts * kCols;
    tile /= kParts;
    set = kMode == kSym && tile >= args.set_tiles ? 1 : 0;
    if (set) tile -= args.set_tiles;
    mat = tile / args.tiles;
    const int t = tile - mat * args.tiles;
    if (kLower) {
      tr = int((sqrtf(8.0f * float(t) + 1.0f) - 1.0f) * 0.5f);
      while ((tr + 1) * (tr + 2) / 2 <= t) ++tr;
      while (tr * (tr + 1) / 2 > t) --tr;
      tc = t - tr * (tr + 1) / 2;
    } else {
      tr = t % args.row_tiles;
      tc = t / args.row_tiles;
    }
  };

  // ---------------- what an epilogue warp does with a 32 x 32 piece of the output --------------
  // A TMEM lane quadrant and a half of the tile's columns per warp.
  const int ew = warp - 2;
  const int quad = warp & 3;
  const int half = ew >> 2;
  const uint32_t lane_addr = tmem_base + (uint32_t(quad * 32) << 16);
  uint8_t* stage_out = staging + ew * kStagingBytes;
  int set = 0, mat = 0, row = 0, row0 = 0;   // of the current tile: this lane's row, the warp's first
  float keep = 0.0f, step = 0.0f;
  // What the epilogue reads is loaded a piece ahead, the first one while the MMAs run, along the
  // rows in memory: of a plane 4 lanes take a row's 64 bytes; of the weights a lane takes a
  // column (of the transposed ones a row).
  uint4 in_v[2][4];
  T w[kPiece];   // as stored: a conversion here would wait for each load before the next
  // final step: this lane's place in the first line of a piece in the caller's matrix (lines are
  // the piece's rows, or its columns where transposed), and how many lines it has there
  auto first_line = [&](int col0, int& lines) {
    const int a = args.transposed ? col0 : row0, b = args.transposed ? row : col0 + lane;
    lines = args.transposed ? (b < args.m ? args.n - a : 0) : (b < args.n ? args.m - a : 0);
    return int64_t(a) * args.out_ld + b;
  };
  auto prefetch = [&](int col0) {
    if constexpr (kMode == kPoly) {
      const int c = col0 + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row0 + i * 8 + (lane >> 2);
        const bool inside = r < args.m && c < int(args.ld);   // ld is a multiple of 8
        const __half* at = args.in + int64_t(mat) * 2 * args.plane + int64_t(r) * args.ld + c;
        in_v[0][i] = inside ? *reinterpret_cast<const uint4*>(at) : make_uint4(0u, 0u, 0u, 0u);
        in_v[1][i] = inside ? *reinterpret_cast<const uint4*>(at + args.plane)
                            : make_uint4(0u, 0u, 0u, 0u);
      }
    } else if constexpr (kMode == kFinal) {
      if (args.has_momentum) {
        int lines;
        const T* p = static_cast<const T*>(outs.p[mat]) + first_line(col0, lines);
#pragma unroll
        for (int k = 0; k < kPiece; ++k, p += args.out_ld)
          if (k < lines) w[k] = *p;
      }
    }
  };
  // The piece at column col0 of the output; next: the column to prefetch then, or -1.
  auto finish = [&](int col0, float (&y)[kPiece], int next) {
    const float mult = args.mult[set];
#pragma unroll
    for (int k = 0; k < kPiece; ++k) y[k] *= mult;
    if constexpr (kMode == kFinal) {
      float o[kPiece];   // element k of this lane's column (transposed: row)
      if (args.transposed) {
#pragma unroll
        for (int k = 0; k < kPiece; ++k) o[k] = y[k];
      } else {
        // through the staging, each word at column XOR row: no two lanes in one bank either way
        float* f = reinterpret_cast<float*>(stage_out);
#pragma unroll
        for (int k = 0; k < kPiece; ++k) f[lane * kPiece + (k ^ lane)] = y[k];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kPiece; ++k) o[k] = f[k * kPiece + (lane ^ k)];
        __syncwarp();
      }
      if (args.has_momentum) {
#pragma unroll
        for (int k = 0; k < kPiece; ++k) o[k] = fmaf(keep, load1(&w[k]), -step * o[k]);
      }
      if (next >= 0) prefetch(next);
      int lines;
      T* p = static_cast<T*>(const_cast<void*>(outs.p[mat])) + first_line(col0, lines);
#pragma unroll
      for (int k = 0; k < kPiece; ++k, p += args.out_ld)
        if (k < lines) *p = from_float<T>(o[k]);
    } else {
      // the planes are ready before the staging's previous store is waited for (poly's: its own
      // input goes through the staging first)
      uint4 h[kPiece / 8], l[kPiece / 8];
      if constexpr (kMode != kPoly) {
#pragma unroll
        for (int g = 0; g < kPiece / 8; ++g) split8(&y[g * 8], h[g], l[g]);
      }
      if (lane == 0) bulk_wait_read();
      __syncwarp();
      if constexpr (kMode == kPoly) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage_out + h * (kStagingBytes / 2) +
                                      plane_offset(i * 8 + (lane >> 2), lane & 3)) = in_v[h][i];
        __syncwarp();
#pragma unroll
        for (int g = 0; g < kPiece / 8; ++g) {
          float x[8];
          join8(*reinterpret_cast<const uint4*>(stage_out + plane_offset(lane, g)),
                *reinterpret_cast<const uint4*>(stage_out + kStagingBytes / 2 +
                                                plane_offset(lane, g)), x);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float& o = y[g * 8 + k];
            o = fmaf(kB, x[k], kC * o);
            if (row == col0 + g * 8 + k) o += kA * kScale;
          }
        }
        __syncwarp();
        if (next >= 0) prefetch(next);
      }
#pragma unroll
      for (int g = 0; g < kPiece / 8; ++g) {
        if constexpr (kMode == kPoly) split8(&y[g * 8], h[g], l[g]);
        *reinterpret_cast<uint4*>(stage_out + plane_offset(lane, g)) = h[g];
        *reinterpret_cast<uint4*>(stage_out + kStagingBytes / 2 + plane_offset(lane, g)) = l[g];
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0 && row0 < args.m && col0 < args.n) {   // TMA leaves out what lies beyond
        const CUtensorMap* out = set ? &tm_out1 : &tm_out0;
        tma_store_3d(out, stage_out, col0, row0, 2 * mat);
        tma_store_3d(out, stage_out + kStagingBytes / 2, col0, row0, 2 * mat + 1);
        bulk_commit();
      }
    }
  };
  constexpr int kPieces = kAccCols / 2 / kPiece;   // of a warp's half of the columns

  if (warp == 0) {
    // ---------------- TMA producer: this CTA's 128 rows of P, its 128 rows or columns of Q ------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, wrapped = false;
      for (int tile = slot0; tile < args.total_tiles && ok; tile += slots) {
        int tset, tmat, tr, tc, part;
        locate(tile, tset, tmat, tr, tc, part);
        const CUtensorMap* tm_q = tset ? &tm_q1 : &tm_q0;
        const int p0 = tr * kTile + int(rank) * kTM, q0 = tc * kTile + part + int(rank) * kTM;
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!wait_phase(empty + stage, phase ^ 1u, abort)) { ok = false; break; }
          uint8_t* s = smem + stage * stage_bytes;
          uint32_t bar = smem_u32(full + stage);
          if constexpr (kPair == 2) bar = cluster_addr(full + stage, 0);
          if (rank == 0) mbar_expect_tx(full + stage, kPair * stage_bytes);
          auto load = [&](void* dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (kPair == 1) tma_load_3d(dst, map, full + stage, x, y, z);
            else tma_load_3d_pair(dst, map, bar, x, y, z);
          };
          const bool mn_p = kSymP && kb * kTK / kTile > tr;
          const bool mn_q = kColsQ || (kSymQ && kb * kTK / kTile > tc);
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {   // boxes of 64 x 64: 64 rows, or 64 columns
              const int p = p0 + b * 64, q = q0 + b * 64, k = kb * kTK;
              load(s + h * kPlaneBytes + b * kBoxBytes, &tm_p, mn_p ? p : k, mn_p ? k : p,
                   2 * tmat + h);
              if (b < kCols / 64)
                load(s + 2 * kPlaneBytes + h * kQBytes + b * kBoxBytes, tm_q, mn_q ? q : k,
                     mn_q ? k : q, 2 * tmat + h);
            }
          }
          if (++stage == stages) { stage = 0; phase ^= 1u; wrapped = true; }
        }
      }
      if (!ok && rank == 0) {
        // given up: the copies in flight land before the block (or the pair) ends
        for (int s = 0; s < stages; ++s)
          if (s < stage || wrapped) drain_phase(full + s, s < stage ? phase : phase ^ 1u);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (rank 0 of a pair issues for both CTAs) ----------------
    // The whole warp walks the tiles, so that what the MMAs take lies in uniform registers.
    if (rank == 0) {
      const uint32_t leader = elect_lane();
      auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, wait_phase(bar, parity, abort)) != 0;
      };
      int stage = 0, local = 0;
      uint32_t phase = 0, used = 0;   // used: how often each accumulator was, modulo 2
      bool issued = false, ok = true;
      auto commit_all = [&](uint64_t* bar) {
        umma_commit<kPair>(kPair == 1 ? smem_u32(bar) : cluster_addr(bar, 0));
        if constexpr (kPair == 2) umma_commit<kPair>(cluster_addr(bar, 1));
      };
      for (int tile = slot0; tile < args.total_tiles && ok; tile += slots, ++local) {
        int tset, tmat, tr, tc, part;
        locate(tile, tset, tmat, tr, tc, part);
        // a sum's first part goes to one accumulator, all others to the other one
        for (int kb0 = 0; kb0 < args.k_blocks && ok; kb0 += args.part_blocks) {
          const int acc = (local & 1) ^ (kb0 != 0 ? 1 : 0);
          if (!wait_warp(tempty + acc, ((used >> acc) & 1) ^ 1u)) { ok = false; break; }
          used ^= 1u << acc;
          tc_fence_after();
          const uint32_t d = tmem_base + uint32_t(acc * kAccCols);
          const int kb1 = min(kb0 + args.part_blocks, args.k_blocks);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!wait_warp(full + stage, phase)) { ok = false; break; }
            tc_fence_after();
            const uint32_t s = smem_u32(smem) + uint32_t(stage) * stage_bytes;
            const bool mn_p = kSymP && __any_sync(0xffffffffu, kb * kTK / kTile > tr);
            const bool mn_q = kColsQ || (kSymQ && __any_sync(0xffffffffu, kb * kTK / kTile > tc));
            auto issue = [&](auto mn_p_, auto mn_q_) {
              issue_block<kPair, kCols, mn_p_.value, mn_q_.value>(
                  d, s, s + 2 * kPlaneBytes, kPlaneBytes, kQBytes, kb != kb0, leader);
            };
            auto issue_q = [&](auto mn_p_) {
              if (mn_q) issue(mn_p_, Const<true>{});
              else issue(mn_p_, Const<false>{});
            };
            if (mn_p) issue_q(Const<true>{});
            else issue_q(Const<false>{});
            issued = true;
            if (leader) commit_all(empty + stage);
            if (++stage == stages) { stage = 0; phase ^= 1u; }
          }
          if (ok && leader) commit_all(tfull + acc);
        }
      }
      if (issued && leader) {
        // Every MMA has completed before the tensor memory is freed.
        umma_commit<kPair>(kPair == 1 ? smem_u32(drain) : cluster_addr(drain, 0));
        drain_phase(drain, 0);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    if (kMode == kFinal && args.has_momentum) {
      const float lr = args.lr_device != nullptr ? *args.lr_device : args.lr;
      keep = 1.0f - lr * args.weight_decay;
      step = lr * args.scale;
    }
    int local = 0;
    uint32_t used = 0;
    auto wait_acc = [&](int acc) {
      const uint32_t parity = (used >> acc) & 1u;
      used ^= 1u << acc;
      int ok = 1;
      if (lane == 0) ok = wait_phase(tfull + acc, parity, abort) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok) (void)mbar_try(tfull + acc, parity);  // completed: acquire for every lane
      tc_fence_after();
      return ok != 0;
    };
    // this warp is done with its part of the accumulator: hand it back to the MMA issuer
    auto hand_back = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair == 1) mbar_arrive(tempty + acc);
        else mbar_arrive_cluster(cluster_addr(tempty + acc, 0));
      }
    };
    for (int tile = slot0; tile < args.total_tiles; tile += slots, ++local) {
      const int acc = local & 1;
      int tr, tc, part;
      locate(tile, set, mat, tr, tc, part);
      row0 = tr * kTile + int(rank) * kTM + quad * 32;
      row = row0 + lane;
      const int col_base = tc * kTile + part + half * (kAccCols / 2);
      prefetch(col_base);
      const uint32_t sums = lane_addr + uint32_t(acc * kAccCols + half * (kAccCols / 2));
      const uint32_t others = lane_addr + uint32_t((acc ^ 1) * kAccCols + half * (kAccCols / 2));
      bool ok = wait_acc(acc);
      for (int kb0 = args.part_blocks; ok && kb0 < args.k_blocks; kb0 += args.part_blocks) {
        ok = wait_acc(acc ^ 1);
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < kPieces; ++c) add_piece(sums + c * kPiece, others + c * kPiece);
        tmem_st_wait();
        hand_back(acc ^ 1);
      }
      if (!ok) break;
#pragma unroll 1
      for (int c = 0; c < kPieces; ++c) {
        float y[kPiece];
        read_piece(sums + c * kPiece, y);
        if (c == kPieces - 1) hand_back(acc);
        const int col0 = col_base + c * kPiece;
        finish(col0, y, c + 1 < kPieces ? col0 + kPiece : -1);
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (kPair == 2) cluster_sync();  // the pair is done with TMEM and remote barriers
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free<kPair>(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// A block of steps on the Gram matrix, m <= 128: one CTA to a matrix.
// ---------------------------------------------------------------------------

struct ChainArgs {
  int32_t m, steps;
};

constexpr int kChainThreads = 512;
// A matrix in shared memory: two planes of two boxes of 128 rows x 64 columns, as TMA swizzles them.
constexpr uint32_t kChainPlane = 2 * kPlaneBytes;
constexpr uint32_t kChainMatrix = 2 * kChainPlane;
constexpr uint32_t kChainSmemBytes = 1024 + 3 * kChainMatrix + 64;
static_assert(kChainSmemBytes <= 227 * 1024, "shared memory");

// Place of the 16-byte granule of columns c .. c + 7 (c a multiple of 8) of row r in a plane.
__device__ __forceinline__ uint32_t chain_offset(int r, int c) {
  return uint32_t(c >> 6) * kPlaneBytes + uint32_t(r) * 128u +
         uint32_t((((c >> 3) & 7) ^ (r & 7)) << 4);
}

// From A to the product Q of the `steps` P's:
//   P = aI + bA + cAA,  Q = P Q (first: P),  A = (P A) P.
// A, P and Q stay in shared memory; every product is complete in tensor memory before its result
// overwrites an operand.  All of them are symmetric, so rows serve as columns throughout.
__global__ void __launch_bounds__(kChainThreads, 1)
kat_muon_chain_kernel(const __grid_constant__ CUtensorMap tm_a,
                      const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ ChainArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* s_a = smem;
  uint8_t* s_p = s_a + kChainMatrix;
  uint8_t* s_q = s_p + kChainMatrix;
  uint64_t* loaded = reinterpret_cast<uint64_t*>(s_q + kChainMatrix);
  uint64_t* done = loaded + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mat = blockIdx.x;
  if (threadIdx.x == 0) {
    mbar_init(loaded, 1);
    mbar_init(done, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tm_a);
    prefetch_map(&tm_q);
  }
  if (warp == 0) tmem_alloc<1>(tmem_slot, kTM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait_previous();

  if (threadIdx.x == 0) {
    // rows and columns behind m arrive as zeros
    mbar_expect_tx(loaded, kChainMatrix);
    for (int h = 0; h < 2; ++h)
      for (int b = 0; b < 4; ++b)
        tma_load_3d(s_a + h * kChainPlane + b * kBoxBytes, &tm_a, loaded, (b >> 1) * 64,
                    (b & 1) * 64, 2 * mat + h);
  }
  auto wait_all = [&](uint64_t* bar, uint32_t parity) {
    int ok = 1;
    if (lane == 0) ok = wait_phase(bar, parity, abort) ? 1 : 0;
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (ok) (void)mbar_try(bar, parity);  // completed: acquire for every lane
    return ok != 0;
  };
  bool ok = __syncthreads_and(wait_all(loaded, 0)) != 0;   // the block gives up together

  // a warp's part of a result: 32 rows, 32 columns
  const int row = (warp & 3) * 32 + lane, col_base = (warp >> 2) * kPiece;
  const uint32_t taddr = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(col_base);
  uint32_t parity = 0;

  // The product of two matrices into tensor memory, complete on return.
  auto product = [&](const uint8_t* p, const uint8_t* q) {
    fence_async_shared();   // the operands were written by this block's threads
    tc_fence_before();      // and the last result has been read
    __syncthreads();
    if (warp == 0 && __all_sync(0xffffffffu, *abort == 0)) {
      const uint32_t leader = elect_lane();
      tc_fence_after();
      const uint32_t sp = smem_u32(p), sq = smem_u32(q);
      issue_block<1, kTM, false, false>(tmem, sp, sq, kChainPlane, kChainPlane, false, leader);
      if (args.m > kTK)
        issue_block<1, kTM, false, false>(tmem, sp + kPlaneBytes, sq + kPlaneBytes, kChainPlane,
                                          kChainPlane, true, leader);
      if (leader) umma_commit<1>(smem_u32(done));
    }
    ok = __syncthreads_and(wait_all(done, parity)) != 0;
    parity ^= 1u;
    tc_fence_after();
  };
  // The result times mult, kept as a matrix in `to` (and `also`); poly: b A + c result + a I.
  auto keep = [&](uint8_t* to, uint8_t* also, float mult, bool poly) {
    float y[kPiece];
    read_piece(taddr, y);
#pragma unroll
    for (int g = 0; g < kPiece / 8; ++g) {
      const int col = col_base + g * 8;
      const uint32_t at = chain_offset(row, col);
      float x[8], v[8];
      if (poly)
        join8(*reinterpret_cast<const uint4*>(s_a + at),
              *reinterpret_cast<const uint4*>(s_a + kChainPlane + at), x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = y[g * 8 + k] * mult;
        if (poly) {
          v[k] = fmaf(kB, x[k], kC * v[k]);
          if (row == col + k) v[k] += kA * kScale;
        }
      }
      uint4 h, l;
      split8(v, h, l);
      *reinterpret_cast<uint4*>(to + at) = h;
      *reinterpret_cast<uint4*>(to + kChainPlane + at) = l;
      if (also != nullptr) {
        *reinterpret_cast<uint4*>(also + at) = h;
        *reinterpret_cast<uint4*>(also + kChainPlane + at) = l;
      }
    }
  };
  const float to_plane = 1.0f / kScale;
  for (int t = 0; t < args.steps && ok; ++t) {
    product(s_a, s_a);
    if (!ok) break;
    keep(s_p, t == 0 ? s_q : nullptr, to_plane, true);
    if (t > 0) {
      product(s_p, s_q);
      if (!ok) break;
      keep(s_q, nullptr, to_plane / 4.0f, false);
    }
    if (t + 1 < args.steps) {
      product(s_p, s_a);
      if (!ok) break;
      keep(s_a, nullptr, to_plane, false);
      product(s_a, s_p);
      if (!ok) break;
      keep(s_a, nullptr, to_plane, false);
    }
  }
  fence_async_shared();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    if (*abort == 0) {
      // Q as it lies: four boxes of 64 x 64, cut at m
      for (int h = 0; h < 2; ++h)
        for (int b = 0; b < 4; ++b)
          if ((b >> 1) * 64 < args.m && (b & 1) * 64 < args.m)
            tma_store_3d(&tm_q, s_q + h * kChainPlane + b * kBoxBytes, (b >> 1) * 64, (b & 1) * 64,
                         2 * mat + h);
      bulk_commit();
      bulk_wait_all();
    } else {
      drain_phase(loaded, 0);   // given up: the copies in flight land before the block ends
    }
  }
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_free<1>(tmem, kTM);
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
// read as zero and not written, so no tile edge needs padding in memory.  `store`: boxes of an
// epilogue warp's 32 x 32 piece instead of an operand's 64 x 64.
bool make_map(CUtensorMap* map, const __half* base, int64_t planes, int64_t rows, int64_t cols,
              int64_t ld, bool store) {
  EncodeTiledFn fn = encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * cuuint64_t(rows) * 2};
  const cuuint32_t box[3] = {store ? cuuint32_t(kPiece) : 64u,
                             store ? cuuint32_t(kPiece) : cuuint32_t(kTK), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
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

// Steps taken on the Gram matrix at once (the blocks of an iteration): wide matrices, whose products
// with X cost more, and those of up to 128 rows, for which a block is one launch.
int block_steps(int64_t m, int64_t n, int left) {
  if (m > kTM && 2 * n < 3 * m) return 1;
  return left == 4 ? 2 : (left < kMaxBlock ? left : kMaxBlock);
}

// Where each part of the workspace lies (bytes; every part a multiple of 256).
struct Layout {
  int64_t m, n, ldn, ldm, plane_x, plane_a;
  size_t x0, x1, sym[6], partial, total;
  Layout(int64_t count, int64_t rows, int64_t cols) {
    m = rows < cols ? rows : cols;
    n = rows < cols ? cols : rows;
    ldn = round_up(n, 8);
    ldm = round_up(m, 8);
    plane_x = m * ldn;
    plane_a = m * ldm;
    const size_t bx = size_t(round_up(count * 2 * plane_x * 2, 256));
    const size_t ba = size_t(round_up(count * 2 * plane_a * 2, 256));
    const int syms = m > kTM && block_steps(m, n, kMaxBlock) > 1 ? 6 : 2;
    x0 = 0;
    x1 = x0 + bx;
    size_t at = x1 + bx;
    for (int i = 0; i < 6; ++i) {
      sym[i] = at;
      if (i < syms) at += ba;
    }
    partial = at;
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

template <typename... Params, typename... Args>
bool launch_after(void (*kernel)(Params...), dim3 grid, int threads, uint32_t smem, int cluster,
                  cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(uint32_t(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = uint32_t(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess;
}

struct Device {
  int sms;
  int pairs;   // CTA pairs that fit at once
};

// Operands and outputs of a product: P, and Q and out of each set.
struct Maps {
  CUtensorMap p, q[2], out[2];
};

template <int kMode, typename T, int kPair, int kCols>
int launch_tiles(const Maps& m, const GemmArgs& args, const PtrTable& outs, int slots,
                cudaStream_t stream) {
  auto kernel = kat_muon_gemm_kernel<kMode, T, kPair, kCols>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(kSmemBytes)) != cudaSuccess)
    return KAT_ERR_CUDA;
  const int grid = args.total_tiles < slots ? args.total_tiles : slots;
  return launch_after(kernel, dim3(uint32_t(grid * kPair)), kThreads, kSmemBytes, kPair, stream,
                      m.p, m.q[0], m.q[1], m.out[0], m.out[1], args, outs)
             ? KAT_OK
             : KAT_ERR_CUDA;
}

// CTA pairs on 256 x 256 tiles, or single CTAs on 128 x 128 tiles?  Of those, halves of 64 columns where
// even these are one wave: a k-block then takes half the MMAs and three quarters of the bytes (one
// [768,768] bf16, 21 to 36 tiles a product: 187 -> 168 us; 3 x [197,1000], 9 to 24 tiles: 180 -> 153).
// What bounds a product then is the planes' way into shared memory, 45 to 50 bytes a cycle of an SM.
template <int kMode, typename T>
int launch_gemm(bool pair, const Maps& m, GemmArgs args, const PtrTable& outs, int sets, int count,
                const Device& dev, cudaStream_t stream) {
  const int side = pair ? 2 * kTM : kTM;
  const int tm = (args.m + side - 1) / side, tn = (args.n + side - 1) / side;
  const int parts = (args.k_blocks + kSumBlocks - 1) / kSumBlocks;
  args.part_blocks = (args.k_blocks + parts - 1) / parts;
  args.row_tiles = tm;
  args.tiles = kMode != kApply && kMode != kFinal ? tm * (tm + 1) / 2 : tm * tn;
  args.set_tiles = args.tiles * count;
  args.total_tiles = args.set_tiles * sets;
  if (pair) return launch_tiles<kMode, T, 2, kTM>(m, args, outs, dev.pairs, stream);
  if (2 * args.total_tiles <= dev.sms) {
    args.total_tiles *= 2;
    return launch_tiles<kMode, T, 1, kTM / 2>(m, args, outs, dev.sms, stream);
  }
  return launch_tiles<kMode, T, 1, kTM>(m, args, outs, dev.sms, stream);
}

template <typename T>
int run(const Update& u, const PtrTable& outs, GemmArgs fin, int32_t count, int64_t rows,
        int64_t cols, int32_t steps, uint8_t* ws, const Device& dev, bool vec,
        cudaStream_t stream) {
  const Layout L(count, rows, cols);
  __half* x[2] = {reinterpret_cast<__half*>(ws + L.x0), reinterpret_cast<__half*>(ws + L.x1)};
  __half* sym[6];
  CUtensorMap mx[2], ms[6], sx[2], ss[6];   // loads and stores of X and of the m x m matrices
  for (int i = 0; i < 2; ++i)
    if (!make_map(&mx[i], x[i], 2 * count, L.m, L.n, L.ldn, false) ||
        !make_map(&sx[i], x[i], 2 * count, L.m, L.n, L.ldn, true))
      return KAT_ERR_CUDA;
  const int syms = L.sym[5] != L.sym[2] ? 6 : 2;
  for (int i = 0; i < syms; ++i) {
    sym[i] = reinterpret_cast<__half*>(ws + L.sym[i]);
    if (!make_map(&ms[i], sym[i], 2 * count, L.m, L.m, L.ldm, false) ||
        !make_map(&ss[i], sym[i], 2 * count, L.m, L.m, L.ldm, true))
      return KAT_ERR_CUDA;
  }
  double* partial = reinterpret_cast<double*>(ws + L.partial);
  const int transposed = rows > cols;

  const int64_t per = int64_t(kNormThreads) * (vec ? 16 : 4);
  const int64_t want = (u.size + per - 1) / per;
  const int norm_blocks = int(want < kNormBlocks ? want : kNormBlocks);
  const dim3 norm_grid{uint32_t(norm_blocks), uint32_t(count)};
  const int row_tiles = int((rows + kSplitTile - 1) / kSplitTile);
  const int col_tiles = int((cols + kSplitTile - 1) / kSplitTile);
  const dim3 split_grid{uint32_t(row_tiles) * uint32_t(col_tiles), uint32_t(count)};
  bool ok;
  if (vec) {
    kat_muon_norm_kernel<T, 8><<<norm_grid, kNormThreads, 0, stream>>>(u, partial);
    ok = launch_after(kat_muon_split_kernel<T, 8>, split_grid, kSplitThreads, 0, 1, stream, u,
                      static_cast<const double*>(partial), norm_blocks, x[0], rows, cols, L.ldn,
                      L.plane_x, transposed, col_tiles);
  } else {
    kat_muon_norm_kernel<T, 1><<<norm_grid, kNormThreads, 0, stream>>>(u, partial);
    ok = launch_after(kat_muon_split_kernel<T, 1>, split_grid, kSplitThreads, 0, 1, stream, u,
                      static_cast<const double*>(partial), norm_blocks, x[0], rows, cols, L.ldn,
                      L.plane_x, transposed, col_tiles);
  }
  if (!ok || cudaGetLastError() != cudaSuccess) return KAT_ERR_CUDA;

  const int k_m = int((L.m + kTK - 1) / kTK), k_n = int((L.n + kTK - 1) / kTK);
  GemmArgs sq{};
  sq.m = sq.n = int32_t(L.m);
  sq.ld = L.ldm;
  sq.plane = L.plane_a;
  sq.k_blocks = k_m;
  sq.mult[0] = 1.0f / kScale;
  fin.m = int32_t(L.m);
  fin.n = int32_t(L.n);
  fin.k_blocks = k_m;
  fin.ld = L.ldn;
  fin.plane = L.plane_x;
  fin.transposed = transposed;
  fin.out_ld = cols;

  // One choice for all products of the call (the symmetric ones store whole tiles of their own size
  // on the diagonal), by the waves of the symmetric ones.
  auto waves = [&](int64_t side, int64_t slots) {
    const int64_t t = (L.m + side - 1) / side;
    return slots > 0 ? (t * (t + 1) / 2 * count + slots - 1) / slots : 0;
  };
  const bool pair = dev.pairs > 0 && 3 * waves(2 * kTM, dev.pairs) <= 2 * waves(kTM, dev.sms);

  // m x m product out0 = p q0, and where q1 >= 0 out1 = p q1 in the same launch
  auto square = [&](int p, int q0, int out0, float mult0, int q1 = -1, int out1 = 0,
                    float mult1 = 0.0f) {
    GemmArgs g = sq;
    const int sets = q1 >= 0 ? 2 : 1;
    g.mult[0] = mult0;
    g.mult[1] = mult1;
    const Maps m{ms[p], {ms[q0], ms[sets == 2 ? q1 : q0]}, {ss[out0], ss[out1]}};
    return launch_gemm<kSym, float>(pair, m, g, outs, sets, count, dev, stream);
  };
  const float to_plane = 1.0f / kScale;
  int cur = 0;
  for (int done = 0; done < steps;) {
    const int block = block_steps(L.m, L.n, steps - done);
    // gram
    GemmArgs g = sq;
    g.k_blocks = k_n;
    const Maps gram{mx[cur], {mx[cur], mx[cur]}, {ss[0], ss[0]}};
    if (int rc = launch_gemm<kGram, float>(pair, gram, g, outs, 1, count, dev, stream)) return rc;
    // sym[0] = A, [1] and [2] the P's in turn, [3] = P A, [4] and [5] the products of P's
    int q = 1;         // where the product of the block's P's so far is
    float q_scale = kScale;
    const bool chained = L.m <= kTM;
    if (chained) {
      const ChainArgs chain{int32_t(L.m), block};
      if (cudaFuncSetAttribute(kat_muon_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               int(kChainSmemBytes)) != cudaSuccess ||
          !launch_after(kat_muon_chain_kernel, dim3(uint32_t(count)), kChainThreads,
                        kChainSmemBytes, 1, stream, ms[0], ms[1], chain))
        return KAT_ERR_CUDA;
      for (int t = 1; t < block; ++t) q_scale /= 4.0f;
    }
    for (int t = chained ? block : 0; t < block; ++t) {
      const int p = 1 + (t & 1);
      g = sq;
      g.in = sym[0];
      const Maps poly{ms[0], {ms[0], ms[0]}, {ss[p], ss[p]}};
      if (int rc = launch_gemm<kPoly, float>(pair, poly, g, outs, 1, count, dev, stream)) return rc;
      const bool more = t + 1 < block;
      const int next = 4 + (t & 1);
      int rc = KAT_OK;
      if (t > 0 && more) rc = square(p, 0, 3, to_plane, q, next, to_plane / 4.0f);
      else if (t > 0) rc = square(p, q, next, to_plane / 4.0f);
      else if (more) rc = square(p, 0, 3, to_plane);
      if (rc) return rc;
      if (t > 0) {
        q = next;
        q_scale /= 4.0f;
      }
      if (more)
        if (int r2 = square(3, p, 0, to_plane)) return r2;
    }
    done += block;
    const Maps apply{ms[q], {mx[cur], mx[cur]}, {sx[cur ^ 1], sx[cur ^ 1]}};
    int rc;
    if (done < steps) {
      fin.mult[0] = 1.0f / q_scale;
      rc = launch_gemm<kApply, float>(pair, apply, fin, outs, 1, count, dev, stream);
    } else {
      fin.mult[0] = 1.0f / (q_scale * kScale);
      rc = launch_gemm<kFinal, T>(pair, apply, fin, outs, 1, count, dev, stream);
    }
    if (rc) return rc;
    cur ^= 1;
  }
  return KAT_OK;
}

// CTA pairs that fit on the current device at once, 0 if none.
int pair_count() {
  auto kernel = kat_muon_gemm_kernel<kApply, float, 2, kTM>;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(kSmemBytes)) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.gridDim = dim3(128);
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
  }
  cudaGetLastError();
  return n;
}

// What the current device `device` holds (asked once).
bool device_of(int device, Device* d) {
  static std::mutex mu;
  static Device cache[64] = {};
  const int sms = sm_count(device);
  if (sms <= 0) return false;
  std::lock_guard<std::mutex> lock(mu);
  if (cache[device].sms == 0) {
    cache[device].pairs = pair_count();
    cache[device].sms = sms;
  }
  *d = cache[device];
  return true;
}

int dispatch(const Update& u, const PtrTable& outs, const GemmArgs& fin, int32_t count,
             int64_t rows, int64_t cols, int32_t dtype, int32_t steps, void* ws, size_t ws_bytes,
             void* stream) {
  const Layout L(count, rows, cols);
  if (ws == nullptr || ws_bytes < L.total || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
    return KAT_ERR_WORKSPACE;
  // tiles of all matrices are counted in 32 bits
  const int64_t tm = (L.m + kTM - 1) / kTM, tn = (L.n + kTM - 1) / kTM;
  if (tm * tn * count >= (int64_t(1) << 30)) return KAT_ERR_BAD_SHAPE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KAT_ERR_CUDA;
  Device d;
  if (!device_of(dev, &d)) return KAT_ERR_CUDA;
  bool vec = cols % 8 == 0;   // the inputs' rows take 16-byte accesses
  for (int i = 0; i < count; ++i)
    vec = vec && ((reinterpret_cast<uintptr_t>(u.x.p[i]) | reinterpret_cast<uintptr_t>(u.m.p[i])) &
                  15u) == 0;
  uint8_t* w = static_cast<uint8_t*>(ws);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case KAT_DTYPE_F32:
      return run<float>(u, outs, fin, count, rows, cols, steps, w, d, vec, st);
    case KAT_DTYPE_F16:
      return run<__half>(u, outs, fin, count, rows, cols, steps, w, d, vec, st);
    default:
      return run<__nv_bfloat16>(u, outs, fin, count, rows, cols, steps, w, d, vec, st);
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
  for (int i = 0; i < count; ++i) {
    if (x[i] == nullptr || out[i] == nullptr) return KAT_ERR_NULL_POINTER;
    u.x.p[i] = x[i];
    outs.p[i] = out[i];
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
  for (int i = 0; i < count; ++i) {
    if (weights[i] == nullptr || grads[i] == nullptr || momenta[i] == nullptr)
      return KAT_ERR_NULL_POINTER;
    u.x.p[i] = grads[i];
    u.m.p[i] = momenta[i];
    outs.p[i] = weights[i];
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
