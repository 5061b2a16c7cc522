// kat_position_bias.cu — learned relative position bias by buckets, forward and backward (C ABI:
// include/kat_position_bias.h).
//
// Distance form.  The bias is constant along diagonals.  Forward: a block looks its diagonals'
// values up once into shared memory; a thread owns 16 bytes of columns and walks down the rows, where its
// window of 16 bytes moves by one: one shared-memory read and a shift for every 16-byte
// store.  Backward: a thread owns 15 neighbouring diagonals and keeps their sums in registers: it
// takes 8 x 8 cells at a time, stepping 8 rows down and 8 columns right, so that every cell is
// read once, in 16-byte accesses, and no two threads add to one sum.  The cells come by cp.async
// into slots of the thread's own, two steps ahead: loads into registers left too few bytes in
// flight (dout[16,4096,4096] bf16: 132 us, 62 % of the copy rate).  Where rows do not start on 16
// bytes, a thread owns one diagonal and a warp reads 32 neighbouring cells of a row.
//
// Index form.  Forward: the table's columns of a few heads in shared memory, cells of the index
// read once for all of them.  Backward: a slab of whole rows goes to shared memory in 16-byte
// accesses; then one thread sums each segment (cells of one bucket, listed by the caller) there.
//
// Both backwards write partial sums that small kernels add in a fixed order: no atomics.

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "kat_rational.h"
#include "kat_position_bias.h"

namespace {

#include "kat_math.cuh"

constexpr int64_t kMaxLength = (int64_t(1) << 31) - 64;

// Read-only loads: the compiler may gather them before the stores to shared memory they alternate with.
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  switch (dtype) {
    case KAT_DTYPE_F32: return __ldg(static_cast<const float*>(p) + i);
    case KAT_DTYPE_F16: return __half2float(__ldg(static_cast<const __half*>(p) + i));
    default: return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
  }
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  switch (dtype) {
    case KAT_DTYPE_F32: static_cast<float*>(p)[i] = v; break;
    case KAT_DTYPE_F16: static_cast<__half*>(p)[i] = __float2half_rn(v); break;
    default: static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); break;
  }
}

// A value's bits in the output type, and those of -infinity.
template <typename T> struct Bits { using U = uint16_t; };
template <> struct Bits<float> { using U = uint32_t; };
template <typename T> __device__ __forceinline__ typename Bits<T>::U bits_of(float v) {
  return Codec<T>::pack1(v);
}

// 16 bytes of neighbouring values of a row: one 16-byte store a thread and row, the lanes next to each
// other (with two stores to a thread, 32 bytes apart from lane to lane, the forward of index[1025,1025],
// 16 heads fp32 took 34 us instead of 24).
template <typename T> constexpr int kCols = 16 / int(sizeof(T));

// ---------------------------------------------------------------------------
// Distance form, forward.
// ---------------------------------------------------------------------------

constexpr int kFwdThreads = 128;

struct DistanceFwd {
  const void* table;
  const int32_t* bucket_of;
  void* out;
  int64_t lq, lk, ld, offset;
  int32_t table_dtype, heads, reach, causal;
  int32_t tx, ty, rows;     // column chunks and row runs of a block, rows of a run
  int32_t col_blocks;
};

template <typename T>
__global__ void __launch_bounds__(kFwdThreads)
kat_distance_bias_fwd_kernel(const __grid_constant__ DistanceFwd a) {
  using U = typename Bits<T>::U;
  extern __shared__ uint32_t fwd_smem[];
  U* f = reinterpret_cast<U*>(fwd_smem);
  const int h = blockIdx.y;
  constexpr int kC = kCols<T>;
  const int64_t j0 = int64_t(blockIdx.x % a.col_blocks) * a.tx * kC;
  const int64_t i0 = int64_t(blockIdx.x / a.col_blocks) * a.ty * a.rows;
  const int span = a.ty * a.rows;
  const int64_t first = j0 - (i0 + span - 1) - a.offset;   // distance of f[0]
  for (int k = threadIdx.x; k < kC * a.tx + span - 1; k += kFwdThreads) {
    const int64_t d = first + k;
    if (a.causal && d > 0) {
      f[k] = bits_of<T>(-__int_as_float(0x7f800000));
    } else {
      const int64_t c = d < -a.reach ? -a.reach : (d > a.reach ? a.reach : d);
      f[k] = bits_of<T>(load_any(a.table, a.table_dtype,
                                 int64_t(__ldg(a.bucket_of + c + a.reach)) * a.heads + h));
    }
  }
  __syncthreads();
  const int tx = threadIdx.x % a.tx, ty = threadIdx.x / a.tx;
  const int64_t j = j0 + kC * tx;
  const int64_t i = i0 + int64_t(ty) * a.rows;
  if (j >= a.ld || i >= a.lq) return;
  // columns behind lk are zero
  uint32_t keep[4], w[4];
  const U* at = f + kC * tx + span - 1 - ty * a.rows;   // (i, j)
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      keep[k] = j + k < a.lk ? 0xffffffffu : 0u;
      w[k] = at[k];
    } else {
      keep[k] = (j + 2 * k < a.lk ? 0xffffu : 0u) | (j + 2 * k + 1 < a.lk ? 0xffff0000u : 0u);
      w[k] = uint32_t(at[2 * k]) | (uint32_t(at[2 * k + 1]) << 16);
    }
  }
  uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t(h) * a.lq + i) * a.ld + j);
  const int64_t step = a.ld / kC;
  const int rows = int(a.lq - i < a.rows ? a.lq - i : a.rows);
  for (int r = 0; r < rows; ++r) {
    *out = make_uint4(w[0] & keep[0], w[1] & keep[1], w[2] & keep[2], w[3] & keep[3]);
    out += step;
    if (r + 1 == rows) break;
    // one row down: every value moves one column right
    const uint32_t next = *--at;
#pragma unroll
    for (int k = 3; k > 0; --k) {
      if constexpr (sizeof(T) == 4) w[k] = w[k - 1];
      else w[k] = __funnelshift_l(w[k - 1], w[k], 16);
    }
    if constexpr (sizeof(T) == 4) w[0] = next;
    else w[0] = (w[0] << 16) | next;
  }
}

// ---------------------------------------------------------------------------
// Distance form, backward.
// ---------------------------------------------------------------------------

constexpr int kBwdThreads = 128;
constexpr int kWin = 16;   // 15 diagonals of a thread, padded
constexpr int kBwdStages = 3;

struct DistanceBwd {
  const void* dout;
  int64_t sh, si, sj;
  int64_t lq, lk, offset;
  int32_t causal, groups;    // groups of 8 rows in a split
  int64_t splits, chunks;    // splits of the rows; threads (windows, or diagonals) of a split
  int64_t threads;           // of all heads and splits
  float* part;               // [head][split][chunk][16], or [head][split][diagonal]
  double* diag;              // [head][lq + lk - 1]
};

template <typename T> __device__ __forceinline__ float load_one(const T* p);
template <> __device__ __forceinline__ float load_one<float>(const float* p) { return __ldg(p); }
template <> __device__ __forceinline__ float load_one<__half>(const __half* p) {
  return __half2float(__ldg(p));
}
template <> __device__ __forceinline__ float load_one<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(__ldg(p));
}

template <typename T> constexpr uint32_t distance_ring_bytes() {
  return uint32_t(kBwdStages) * kBwdThreads * 64 * uint32_t(sizeof(T));
}

// Rows start on 16 bytes: a thread owns the diagonals 8c - 7 .. 8c + 7.
template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
kat_distance_bias_bwd_kernel(const __grid_constant__ DistanceBwd a) {
  constexpr int kWords = int(sizeof(T)) / 2;   // 16-byte words of 8 cells
  extern __shared__ uint4 cell_smem[];
  const int64_t id = int64_t(blockIdx.x) * kBwdThreads + threadIdx.x;
  if (id >= a.threads) return;
  const int64_t k = id % a.chunks, split = id / a.chunks % a.splits, h = id / a.chunks / a.splits;
  const int64_t g0 = split * a.groups;
  const int64_t rows8 = (a.lq + 7) / 8, cols8 = (a.lk + 7) / 8;
  const int64_t g1 = g0 + a.groups < rows8 ? g0 + a.groups : rows8;
  const int64_t c = k - (g0 + a.groups - 1);
  if (a.causal && 8 * c - 7 > a.offset) return;     // masked, and never read
  float acc[15], tot[15];   // 256 terms at most go one after the other into a sum
#pragma unroll
  for (int i = 0; i < 15; ++i) acc[i] = tot[i] = 0.0f;
  const T* base = static_cast<const T*>(a.dout) + h * a.sh;
  const int64_t gb = g0 > -c ? g0 : -c, ge = g1 < cols8 - c ? g1 : cols8 - c;
  // of the steps gb .. ge - 1 only the last may reach over the last row or column
  int64_t whole = a.lq / 8 < a.lk / 8 - c ? a.lq / 8 : a.lk / 8 - c;
  if (whole > ge) whole = ge;
  const int steps = whole > gb ? int(whole - gb) : 0;
  const uint32_t slot0 =
      static_cast<uint32_t>(__cvta_generic_to_shared(cell_smem)) + threadIdx.x * 16u;
  auto slot = [&](int stage, int r, int q) {
    return slot0 + uint32_t(((stage * 8 + r) * kWords + q) * kBwdThreads * 16);
  };
  const T* next = base + gb * 8 * a.si + (c + gb) * 8;
  int left = steps;
  auto fetch = [&](int stage) {
    if (left > 0) {
      --left;
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < kWords; ++q)
          asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(slot(stage, r, q)),
                       "l"(next + r * a.si + q * (16 / int(sizeof(T)))) : "memory");
      next += 8 * a.si + 8;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kBwdStages - 1; ++i) fetch(i);
  int stage = 0;
  for (int t = 0; t < steps; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kBwdStages - 2) : "memory");
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
      for (int q = 0; q < kWords; ++q) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(slot(stage, r, q))
                     : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            acc[4 * q + e - r + 7] += __uint_as_float(w[e]);
          } else {
            const float2 v = Codec<T>::unpack_word(w[e]);
            acc[2 * e - r + 7] += v.x;
            acc[2 * e + 1 - r + 7] += v.y;
          }
        }
      }
    }
    fetch(stage == 0 ? kBwdStages - 1 : stage - 1);
    if (++stage == kBwdStages) stage = 0;
    if ((t & 31) == 31) {
#pragma unroll
      for (int i = 0; i < 15; ++i) {
        tot[i] += acc[i];
        acc[i] = 0.0f;
      }
    }
  }
  for (int64_t g = gb + steps; g < ge; ++g) {
    const T* p = base + 8 * g * a.si + 8 * (c + g);
    const int64_t rows = a.lq - 8 * g, cols = a.lk - 8 * (c + g);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (r < rows && e < cols) acc[e - r + 7] += load_one(p + e);
      p += a.si;
      asm volatile("" ::: "memory");   // one row's loads at a time: 64 would fill the registers
    }
  }
#pragma unroll
  for (int i = 0; i < 15; ++i) acc[i] += tot[i];
  float4* to = reinterpret_cast<float4*>(a.part + id * kWin);
  to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  to[2] = make_float4(acc[8], acc[9], acc[10], acc[11]);
  to[3] = make_float4(acc[12], acc[13], acc[14], 0.0f);
}

// Any strides: a thread owns one diagonal.
template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
kat_distance_bias_bwd_any_kernel(const __grid_constant__ DistanceBwd a) {
  const int64_t id = int64_t(blockIdx.x) * kBwdThreads + threadIdx.x;
  if (id >= a.threads) return;
  const int64_t k = id % a.chunks, split = id / a.chunks % a.splits, h = id / a.chunks / a.splits;
  const int64_t d = k - (a.lq - 1);
  if (a.causal && d > a.offset) return;
  int64_t i0 = split * a.groups * 8, i1 = i0 + int64_t(a.groups) * 8;
  if (i0 < -d) i0 = -d;
  if (i1 > a.lq) i1 = a.lq;
  if (i1 > a.lk - d) i1 = a.lk - d;
  const int64_t step = a.si + a.sj;
  const T* p = static_cast<const T*>(a.dout) + h * a.sh + i0 * a.si + (i0 + d) * a.sj;
  float total = 0.0f;
  while (i0 < i1) {
    const int64_t end = i0 + 256 < i1 ? i0 + 256 : i1;
    float sum = 0.0f;
#pragma unroll 8
    for (; i0 < end; ++i0, p += step) sum += load_one(p);
    total += sum;
  }
  a.part[id] = total;
}

// One sum for each diagonal: its splits, in each of which two windows hold it (kVec) or one thread.
// 32 diagonals to a block, their splits in 8 runs added in order.
template <bool kVec>
__global__ void __launch_bounds__(256)
kat_distance_bias_diag_kernel(const __grid_constant__ DistanceBwd a) {
  const int64_t count = a.lq + a.lk - 1;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t k = int64_t(blockIdx.x) * 32 + tx;
  const int64_t h = blockIdx.y;
  const int64_t d = k - (a.lq - 1);
  double sum = 0.0;
  if (k < count && (!a.causal || d <= a.offset)) {
    // from split to split: the next part, and there the window that lies `groups` further
    const float* part = a.part + (h * a.splits + ty) * a.chunks * (kVec ? kWin : 1);
    const int splits = int(a.splits);
    if constexpr (kVec) {
      const int c = int(d >= 0 ? d / 8 : -((7 - d) / 8)), o = int(d - 8 * int64_t(c));
      const int chunks = int(a.chunks);
      int at = c + ty * a.groups + a.groups - 1;
      const float* p = part + int64_t(at) * kWin + o;
      const int64_t step = 8 * (a.chunks + a.groups) * kWin;
#pragma unroll 2
      for (int s = ty; s < splits; s += 8, at += 8 * a.groups, p += step) {
        const float one = unsigned(at) < unsigned(chunks) ? p[7] : 0.0f;
        const float two = o > 0 && unsigned(at + 1) < unsigned(chunks) ? p[kWin - 1] : 0.0f;
        sum += double(one) + double(two);
      }
    } else {
      const float* p = part + k;
#pragma unroll 4
      for (int s = ty; s < splits; s += 8, p += 8 * a.chunks) sum += double(*p);
    }
  }
  __shared__ double acc[8][32];
  acc[ty][tx] = sum;
  __syncthreads();
  if (ty == 0 && k < count) {
#pragma unroll
    for (int r = 1; r < 8; ++r) sum += acc[r][tx];
    a.diag[h * count + k] = sum;
  }
}

// A bucket's run of diagonals, one block.
__global__ void __launch_bounds__(256)
kat_distance_bias_run_kernel(const __grid_constant__ DistanceBwd a,
                             const int32_t* __restrict__ run_begin,
                             const int32_t* __restrict__ run_end, int heads, void* d_table,
                             int table_dtype) {
  const int b = blockIdx.x, h = blockIdx.y;
  const int64_t low = -(a.lq - 1), high = a.lk - 1;
  int64_t begin = run_begin[b], end = run_end[b];
  begin = begin == INT32_MIN ? low : begin + a.offset;
  end = end == INT32_MAX ? high : end + a.offset;
  if (begin < low) begin = low;
  if (end > high) end = high;
  const double* diag = a.diag + int64_t(h) * (a.lq + a.lk - 1) + (a.lq - 1);
  double sum = 0.0;
  for (int64_t d = begin + threadIdx.x; d <= end; d += 256) sum += diag[d];
  __shared__ double acc[8];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if ((threadIdx.x & 31) == 0) acc[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) sum += acc[w];
    store_any(d_table, table_dtype, int64_t(b) * heads + h, float(sum));
  }
}

// ---------------------------------------------------------------------------
// Index form.
// ---------------------------------------------------------------------------

constexpr int kIdxThreads = 256;
constexpr int kIdxBwdThreads = 512;
constexpr int kIdxSmem = 64 * 1024;       // table columns of a block
constexpr int kIdxSmemMost = 200 * 1024;  // above this even one column stays in global memory

struct IndexFwd {
  const void* table;
  const int32_t* index;
  void* out;
  int64_t chunks;          // lq * ld cells, 16 bytes of the output to a chunk
  int32_t table_dtype, num_buckets, heads;
  int32_t group;           // heads of a block
};

// Neighbouring cells of a grid's row have neighbouring buckets, a power of two apart from lane to lane:
// one place more every 32 keeps them in different banks.
__device__ __forceinline__ int spread(int b) { return b + (b >> 5); }

template <typename T, bool kSmem>
__global__ void __launch_bounds__(kIdxThreads)
kat_index_bias_fwd_kernel(const __grid_constant__ IndexFwd a) {
  using U = typename Bits<T>::U;
  extern __shared__ uint32_t idx_smem[];
  U* f = reinterpret_cast<U*>(idx_smem);
  const int h0 = blockIdx.y * a.group;
  const int heads = a.heads - h0 < a.group ? a.heads - h0 : a.group;
  const int pitch = spread(a.num_buckets) + 1;   // the last one is the zero of cells without bias
  if constexpr (kSmem) {
    // table rows four at a time, four of their heads each, all loads before the stores
    for (int b0 = threadIdx.x; b0 < a.num_buckets; b0 += 4 * kIdxThreads) {
      for (int g = 0; g < heads; g += 4) {
        float v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int b = b0 + i * kIdxThreads;
            v[i][h] = b < a.num_buckets && g + h < heads
                          ? load_any(a.table, a.table_dtype, int64_t(b) * a.heads + h0 + g + h)
                          : 0.0f;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int b = b0 + i * kIdxThreads;
            if (b < a.num_buckets && g + h < heads) f[(g + h) * pitch + spread(b)] = bits_of<T>(v[i][h]);
          }
      }
    }
    for (int h = threadIdx.x; h < heads; h += kIdxThreads)
      f[h * pitch + spread(a.num_buckets)] = U(0);
    __syncthreads();
  }
  for (int64_t k = int64_t(blockIdx.x) * kIdxThreads + threadIdx.x; k < a.chunks;
       k += int64_t(gridDim.x) * kIdxThreads) {
    constexpr int kC = kCols<T>;
    int at[kC];
#pragma unroll
    for (int q = 0; q < kC / 4; ++q) {
      const int4 v = __ldg(reinterpret_cast<const int4*>(a.index) + k * (kC / 4) + q);
      at[4 * q] = v.x;
      at[4 * q + 1] = v.y;
      at[4 * q + 2] = v.z;
      at[4 * q + 3] = v.w;
    }
    if constexpr (kSmem) {
#pragma unroll
      for (int e = 0; e < kC; ++e) at[e] = spread(at[e]);
    }
    for (int h = 0; h < heads; ++h) {
      uint32_t v[kC];
#pragma unroll
      for (int e = 0; e < kC; ++e) {
        if constexpr (kSmem) {
          v[e] = f[h * pitch + at[e]];
        } else {
          v[e] = at[e] == a.num_buckets
                     ? 0u
                     : uint32_t(bits_of<T>(load_any(a.table, a.table_dtype,
                                                    int64_t(at[e]) * a.heads + h0 + h)));
        }
      }
      uint4* out = reinterpret_cast<uint4*>(a.out) + int64_t(h0 + h) * a.chunks + k;
      if constexpr (sizeof(T) == 4)
        *out = make_uint4(v[0], v[1], v[2], v[3]);
      else
        *out = make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16),
                          v[6] | (v[7] << 16));
    }
  }
}

struct IndexBwd {
  const void* dout;
  int64_t sh, si, sj;
  int64_t lq, lk, pitch;   // pitch: cells from row to row in `cells`
  const uint16_t* cells;
  const int32_t* seg_begin;
  const int32_t* slab_begin;
  const int32_t* seg_place;
  int64_t segments;
  int32_t slab_rows, slab_bytes;
  int32_t heads, group;    // heads in all, and of a block
  float* part;             // [head][place of the segment]
};

// kFlat: the slab's rows are one run of memory of the cells' own pitch, which goes to shared memory
// as it lies there: every 16 bytes on a 16-byte boundary by cp.async, all of them in flight at
// once, and the cells are read `skew` places further.  (Spreading pieces from registers over padded
// rows instead cost four times the shared-memory wavefronts: dout[16,1025,1025] fp32 61 us.)
// Otherwise cell by cell, into rows of the cells' pitch.
// The list of the slab's cells goes to shared memory too, once for the block's heads.
template <typename T, bool kFlat>
__global__ void __launch_bounds__(kIdxBwdThreads)
kat_index_bias_bwd_kernel(const __grid_constant__ IndexBwd a) {
  using U = typename Bits<T>::U;
  extern __shared__ uint4 slab_smem[];
  uint4* list_smem = slab_smem + a.slab_bytes / 16;
  const int64_t i0 = int64_t(blockIdx.x) * a.slab_rows;
  const uint32_t rows = uint32_t(a.lq - i0 < a.slab_rows ? a.lq - i0 : a.slab_rows);
  const uint32_t pitch = uint32_t(a.pitch), lk = uint32_t(a.lk);
  const int32_t seg_first = __ldg(a.slab_begin + blockIdx.x);
  const int32_t seg_end = __ldg(a.slab_begin + blockIdx.x + 1);
  const int32_t cell_first = __ldg(a.seg_begin + seg_first);
  const uint16_t* list;
  // `count` elements from `from` into `to`, as they lie: the place of the first one there
  auto copy_run = [&](auto* to_raw, const auto* from, uint32_t count) {
    constexpr uint32_t kPer = 16 / sizeof(*from);
    const uint32_t skew = uint32_t(reinterpret_cast<uintptr_t>(from) & 15u) / sizeof(*from);
    auto* to = to_raw;
    const uint32_t to0 = static_cast<uint32_t>(__cvta_generic_to_shared(to_raw));
    for (uint32_t k = threadIdx.x; k * kPer < count + skew; k += kIdxBwdThreads) {
      const int32_t first = int32_t(k * kPer) - int32_t(skew);   // the piece's first element
      if (first >= 0 && first + kPer <= count) {
        asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(to0 + k * 16u),
                     "l"(from + first) : "memory");
      } else {   // the run's ends
        for (uint32_t e = 0; e < kPer; ++e)
          if (first + int32_t(e) >= 0 && first + e < count)
            to[k * kPer + e] = __ldg(from + first + e);
      }
    }
    return to + skew;
  };
  list = copy_run(reinterpret_cast<uint16_t*>(list_smem), a.cells + cell_first,
                  uint32_t(__ldg(a.seg_begin + seg_end) - cell_first));
  const int h0 = blockIdx.y * a.group;
  const int h1 = h0 + a.group < a.heads ? h0 + a.group : a.heads;
  for (int64_t h = h0; h < h1; ++h) {
    const U* base = static_cast<const U*>(a.dout) + h * a.sh + i0 * a.si;
    const U* s = reinterpret_cast<const U*>(slab_smem);
    if constexpr (kFlat) {
      s = copy_run(reinterpret_cast<U*>(slab_smem), base, (rows - 1) * pitch + lk);
    } else {
      U* to = reinterpret_cast<U*>(slab_smem);
      for (uint32_t k = threadIdx.x; k < rows * lk; k += kIdxBwdThreads) {
        const uint32_t r = k / lk, j = k % lk;
        to[r * pitch + j] = __ldg(base + int64_t(r) * a.si + int64_t(j) * a.sj);
      }
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    for (int32_t g = seg_first + int(threadIdx.x); g < seg_end; g += kIdxBwdThreads) {
      float sum = 0.0f;
      const int32_t place = __ldg(a.seg_place + g);
      const int32_t last = __ldg(a.seg_begin + g + 1) - cell_first;
#pragma unroll 4
      for (int32_t k = __ldg(a.seg_begin + g) - cell_first; k < last; ++k)
        sum += Codec<T>::unpack1(s[list[k]]);
      a.part[h * a.segments + place] = sum;
    }
    __syncthreads();
  }
}

// The segments of a bucket for one head, by 8 lanes.
__global__ void __launch_bounds__(256)
kat_index_bias_bucket_kernel(const float* __restrict__ part, int64_t segments,
                             const int32_t* __restrict__ bucket_begin, int num_buckets, int heads,
                             void* d_table, int table_dtype) {
  const int64_t k = int64_t(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const int lane = threadIdx.x & 7;
  const bool live = k < int64_t(num_buckets) * heads;
  const int b = live ? int(k % num_buckets) : 0, h = live ? int(k / num_buckets) : 0;
  double sum = 0.0;
  if (live) {
    const int32_t end = bucket_begin[b + 1];
#pragma unroll 4
    for (int32_t g = bucket_begin[b] + lane; g < end; g += 8)
      sum += double(part[int64_t(h) * segments + g]);
  }
#pragma unroll
  for (int m = 4; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (live && lane == 0) store_any(d_table, table_dtype, int64_t(b) * heads + h, float(sum));
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

bool known(int dtype) {
  return dtype == KAT_DTYPE_F32 || dtype == KAT_DTYPE_F16 || dtype == KAT_DTYPE_BF16;
}
int elem_size(int dtype) { return dtype == KAT_DTYPE_F32 ? 4 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

int check_common(int32_t a_dtype, int32_t b_dtype, int32_t num_buckets, int32_t heads, int64_t lq,
                 int64_t lk) {
  if (!known(a_dtype) || !known(b_dtype)) return KAT_ERR_BAD_DTYPE;
  if (num_buckets < 1 || num_buckets > (1 << 24) || heads < 0 || heads > 65535 || lq < 0 ||
      lk < 0 || lq > kMaxLength || lk > kMaxLength)
    return KAT_ERR_BAD_SHAPE;
  return KAT_OK;
}

// Whether rows of a gradient can be read in 16-byte pieces.
bool vector_rows(const void* p, int dtype, const int64_t* stride) {
  const int per = 16 / elem_size(dtype);
  return aligned16(p) && stride[2] == 1 && stride[1] % per == 0 && stride[0] % per == 0;
}

struct DistancePlan {
  int32_t groups;
  int64_t splits, chunks;
  size_t part, total;
};
// Groups of 8 rows in a split: the most that leave the device about two waves of blocks (4 of
// windows or 16 of diagonals to an SM).  dout[16,4096,4096] bf16, kernel and sum over the splits:
// 8 groups 99 + 37 us, 16: 101 + 19, 32: 103 + 11, 64 (one wave, its blocks of unequal length):
// 125 + 6; the sum over the splits has since become quicker.
DistancePlan distance_plan(int32_t heads, int64_t lq, int64_t lk, bool vec) {
  const int64_t rows8 = (lq + 7) / 8, cols8 = (lk + 7) / 8;
  const double resident = 148.0 * kBwdThreads * (vec ? 4 : 16);
  auto splits = [&](int64_t n) { return (rows8 + n - 1) / n; };
  auto chunks = [&](int64_t n) { return vec ? cols8 + n - 1 : lq + lk - 1; };
  int64_t g = 1024;
  while (g > 1 && double(heads) * double(splits(g)) * double(chunks(g)) < 1.75 * resident) g /= 2;
  DistancePlan p;
  p.groups = int32_t(g);
  p.splits = splits(g);
  p.chunks = chunks(g);
  p.part = size_t(heads) * size_t(p.splits) * size_t(p.chunks) * (vec ? kWin : 1) * sizeof(float);
  p.part = (p.part + 15) / 16 * 16;
  p.total = p.part + size_t(heads) * size_t(lq + lk - 1) * sizeof(double);
  return p;
}

template <typename K>
int set_smem(K kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return KAT_OK;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) ==
                 cudaSuccess
             ? KAT_OK
             : KAT_ERR_CUDA;
}
int launched() { return cudaGetLastError() == cudaSuccess ? KAT_OK : KAT_ERR_CUDA; }

template <typename T>
void launch_distance_fwd(const DistanceFwd& a, dim3 grid, size_t smem, cudaStream_t st) {
  kat_distance_bias_fwd_kernel<T><<<grid, kFwdThreads, smem, st>>>(a);
}

template <typename T>
int launch_distance_bwd(const DistanceBwd& a, bool vec, dim3 grid, cudaStream_t st) {
  if (!vec) {
    kat_distance_bias_bwd_any_kernel<T><<<grid, kBwdThreads, 0, st>>>(a);
    return launched();
  }
  constexpr uint32_t bytes = distance_ring_bytes<T>();
  if (int rc = set_smem(kat_distance_bias_bwd_kernel<T>, bytes)) return rc;
  kat_distance_bias_bwd_kernel<T><<<grid, kBwdThreads, bytes, st>>>(a);
  return launched();
}

template <typename T>
int launch_index_fwd(IndexFwd a, cudaStream_t st) {
  const size_t column = size_t(a.num_buckets + (a.num_buckets >> 5) + 1) * sizeof(T);
  const bool smem = column <= size_t(kIdxSmemMost);
  int group = smem ? int(size_t(kIdxSmem) / column) : a.heads;
  if (group < 1) group = 1;
  if (group > a.heads) group = a.heads;
  int64_t blocks = (a.chunks + kIdxThreads - 1) / kIdxThreads;
  // small indices: fewer heads to a block, until the blocks fill the device
  while (group > 1 && blocks * ((a.heads + group - 1) / group) < 148 * 2) group = (group + 1) / 2;
  a.group = group;
  const int head_blocks = (a.heads + group - 1) / group;
  // large ones: a block loads its table columns once and takes several runs of cells, as many as
  // make one wave of blocks (index[1025,1025], 16 heads fp32: six waves spent 69 us, most of it on
  // the columns)
  const int64_t most = (148 * (smem ? 3 : 8) + head_blocks - 1) / head_blocks;
  if (blocks > most) blocks = most;
  const dim3 grid{uint32_t(blocks), uint32_t(head_blocks)};
  if (smem) {
    const size_t bytes = (column * group + 3) / 4 * 4;
    if (int rc = set_smem(kat_index_bias_fwd_kernel<T, true>, bytes)) return rc;
    kat_index_bias_fwd_kernel<T, true><<<grid, kIdxThreads, bytes, st>>>(a);
  } else {
    kat_index_bias_fwd_kernel<T, false><<<grid, kIdxThreads, 0, st>>>(a);
  }
  return launched();
}

template <typename T, bool kFlat>
int launch_index_bwd_v(IndexBwd a, int64_t slabs, cudaStream_t st) {
  const size_t cells = size_t(a.slab_rows) * size_t(a.pitch);
  a.slab_bytes = int32_t((cells * sizeof(T) + 16 + 15) / 16 * 16);   // a run may start 15 bytes in
  const size_t bytes = size_t(a.slab_bytes) + cells * 2 + 16;
  // as many heads to a block as leave two blocks for every SM
  a.group = 1;
  while (a.group < a.heads && slabs * ((a.heads + 2 * a.group - 1) / (2 * a.group)) >= 2 * 148)
    a.group *= 2;
  if (int rc = set_smem(kat_index_bias_bwd_kernel<T, kFlat>, bytes)) return rc;
  const dim3 grid{uint32_t(slabs), uint32_t((a.heads + a.group - 1) / a.group)};
  kat_index_bias_bwd_kernel<T, kFlat><<<grid, kIdxBwdThreads, bytes, st>>>(a);
  return launched();
}
template <typename T>
int launch_index_bwd(const IndexBwd& a, int64_t slabs, cudaStream_t st) {
  return a.sj == 1 && a.si == a.pitch ? launch_index_bwd_v<T, true>(a, slabs, st)
                                      : launch_index_bwd_v<T, false>(a, slabs, st);
}

}  // namespace

extern "C" {

int kat_distance_bias_fwd(const void* table, int32_t table_dtype, int32_t num_buckets,
                          int32_t heads, const int32_t* bucket_of, int32_t reach, int64_t lq,
                          int64_t lk, int64_t offset, int32_t causal, void* out,
                          int32_t out_dtype, void* stream) {
  if (int rc = check_common(table_dtype, out_dtype, num_buckets, heads, lq, lk)) return rc;
  if (reach < 0 || offset > kMaxLength || offset < -kMaxLength) return KAT_ERR_BAD_SHAPE;
  if (heads == 0 || lq == 0 || lk == 0) return KAT_OK;
  if (table == nullptr || bucket_of == nullptr || out == nullptr) return KAT_ERR_NULL_POINTER;
  if (!aligned16(out)) return KAT_ERR_BAD_SHAPE;
  DistanceFwd a{};
  a.table = table;
  a.bucket_of = bucket_of;
  a.out = out;
  a.lq = lq;
  a.lk = lk;
  a.ld = round8(lk);
  a.offset = offset;
  a.table_dtype = table_dtype;
  a.heads = heads;
  a.reach = reach;
  a.causal = causal != 0;
  const int per = 16 / elem_size(out_dtype);   // columns of a thread
  const int64_t chunks = a.ld / per;
  a.tx = 1;
  while (a.tx < kFwdThreads && a.tx < chunks) a.tx *= 2;
  a.ty = kFwdThreads / a.tx;
  const int64_t col_blocks = (chunks + a.tx - 1) / a.tx;
  auto blocks = [&](int64_t rows) {
    return col_blocks * ((lq + a.ty * rows - 1) / (a.ty * rows));
  };
  // long runs amortise the lookups; short ones fill the device
  a.rows = 32;
  while (a.rows > 1 && blocks(a.rows) * heads < 148 * 8) a.rows /= 2;
  const int64_t n = blocks(a.rows);
  if (n >= (int64_t(1) << 31) || col_blocks >= (int64_t(1) << 31)) return KAT_ERR_BAD_SHAPE;
  a.col_blocks = int32_t(col_blocks);
  const size_t smem =
      (size_t(per * a.tx + a.ty * a.rows - 1) * elem_size(out_dtype) + 3) / 4 * 4;
  const dim3 grid{uint32_t(n), uint32_t(heads)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case KAT_DTYPE_F32: launch_distance_fwd<float>(a, grid, smem, st); break;
    case KAT_DTYPE_F16: launch_distance_fwd<__half>(a, grid, smem, st); break;
    default: launch_distance_fwd<__nv_bfloat16>(a, grid, smem, st); break;
  }
  return launched();
}

size_t kat_distance_bias_bwd_workspace_bytes(int32_t heads, int64_t lq, int64_t lk) {
  if (check_common(KAT_DTYPE_F32, KAT_DTYPE_F32, 1, heads, lq, lk) != KAT_OK || heads == 0 ||
      lq == 0 || lk == 0)
    return 0;
  const size_t vec = distance_plan(heads, lq, lk, true).total;
  const size_t any = distance_plan(heads, lq, lk, false).total;
  return vec > any ? vec : any;
}

int kat_distance_bias_bwd(const void* dout, int32_t dout_dtype, const int64_t* dout_stride,
                          int32_t num_buckets, int32_t heads, const int32_t* run_begin,
                          const int32_t* run_end, int64_t lq, int64_t lk, int64_t offset,
                          int32_t causal, void* d_table, int32_t table_dtype, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (int rc = check_common(table_dtype, dout_dtype, num_buckets, heads, lq, lk)) return rc;
  if (offset > kMaxLength || offset < -kMaxLength) return KAT_ERR_BAD_SHAPE;
  if (heads == 0) return KAT_OK;
  if (d_table == nullptr) return KAT_ERR_NULL_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (lq == 0 || lk == 0)  // sums over no cells
    return cudaMemsetAsync(d_table, 0, size_t(num_buckets) * heads * elem_size(table_dtype), st) ==
                   cudaSuccess
               ? KAT_OK
               : KAT_ERR_CUDA;
  if (dout == nullptr || dout_stride == nullptr || run_begin == nullptr || run_end == nullptr)
    return KAT_ERR_NULL_POINTER;
  const bool vec = vector_rows(dout, dout_dtype, dout_stride);
  const DistancePlan plan = distance_plan(heads, lq, lk, vec);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < plan.total)
    return KAT_ERR_WORKSPACE;
  DistanceBwd a{};
  a.dout = dout;
  a.sh = dout_stride[0];
  a.si = dout_stride[1];
  a.sj = dout_stride[2];
  a.lq = lq;
  a.lk = lk;
  a.offset = offset;
  a.causal = causal != 0;
  a.groups = plan.groups;
  a.splits = plan.splits;
  a.chunks = plan.chunks;
  a.threads = int64_t(heads) * plan.splits * plan.chunks;
  a.part = static_cast<float*>(workspace);
  a.diag = reinterpret_cast<double*>(static_cast<uint8_t*>(workspace) + plan.part);
  const int64_t blocks = (a.threads + kBwdThreads - 1) / kBwdThreads;
  if (blocks >= (int64_t(1) << 31)) return KAT_ERR_BAD_SHAPE;
  const dim3 grid{uint32_t(blocks)};
  int rc = KAT_OK;
  switch (dout_dtype) {
    case KAT_DTYPE_F32: rc = launch_distance_bwd<float>(a, vec, grid, st); break;
    case KAT_DTYPE_F16: rc = launch_distance_bwd<__half>(a, vec, grid, st); break;
    default: rc = launch_distance_bwd<__nv_bfloat16>(a, vec, grid, st); break;
  }
  if (rc) return rc;
  const dim3 diag_grid{uint32_t((lq + lk - 1 + 31) / 32), uint32_t(heads)};
  if (vec) kat_distance_bias_diag_kernel<true><<<diag_grid, 256, 0, st>>>(a);
  else kat_distance_bias_diag_kernel<false><<<diag_grid, 256, 0, st>>>(a);
  kat_distance_bias_run_kernel<<<dim3(uint32_t(num_buckets), uint32_t(heads)), 256, 0, st>>>(
      a, run_begin, run_end, heads, d_table, table_dtype);
  return launched();
}

int kat_index_bias_fwd(const void* table, int32_t table_dtype, int32_t num_buckets, int32_t heads,
                       const int32_t* index, int64_t lq, int64_t lk, void* out, int32_t out_dtype,
                       void* stream) {
  if (int rc = check_common(table_dtype, out_dtype, num_buckets, heads, lq, lk)) return rc;
  if (heads == 0 || lq == 0 || lk == 0) return KAT_OK;
  if (table == nullptr || index == nullptr || out == nullptr) return KAT_ERR_NULL_POINTER;
  if (!aligned16(out) || !aligned16(index)) return KAT_ERR_BAD_SHAPE;
  IndexFwd a{};
  a.table = table;
  a.index = index;
  a.out = out;
  a.chunks = lq * (round8(lk) / (16 / elem_size(out_dtype)));
  a.table_dtype = table_dtype;
  a.num_buckets = num_buckets;
  a.heads = heads;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case KAT_DTYPE_F32: return launch_index_fwd<float>(a, st);
    case KAT_DTYPE_F16: return launch_index_fwd<__half>(a, st);
    default: return launch_index_fwd<__nv_bfloat16>(a, st);
  }
}

size_t kat_index_bias_bwd_workspace_bytes(int32_t heads, int64_t segments) {
  if (heads < 0 || segments < 0) return 0;
  return size_t(heads) * size_t(segments) * sizeof(float);
}

int kat_index_bias_bwd(const void* dout, int32_t dout_dtype, const int64_t* dout_stride,
                       int32_t num_buckets, int32_t heads, int64_t lq, int64_t lk,
                       const uint16_t* cells, const uint16_t* padded_cells,
                       const int32_t* seg_begin, int64_t segments, const int32_t* slab_begin,
                       int64_t slabs, int32_t slab_rows,
                       const int32_t* seg_place, const int32_t* bucket_begin, void* d_table,
                       int32_t table_dtype, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (int rc = check_common(table_dtype, dout_dtype, num_buckets, heads, lq, lk)) return rc;
  if (heads == 0) return KAT_OK;
  if (d_table == nullptr) return KAT_ERR_NULL_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (lq == 0 || lk == 0 || segments == 0)
    return cudaMemsetAsync(d_table, 0, size_t(num_buckets) * heads * elem_size(table_dtype), st) ==
                   cudaSuccess
               ? KAT_OK
               : KAT_ERR_CUDA;
  if (dout == nullptr || dout_stride == nullptr || cells == nullptr || padded_cells == nullptr ||
      seg_begin == nullptr ||
      slab_begin == nullptr || seg_place == nullptr || bucket_begin == nullptr)
    return KAT_ERR_NULL_POINTER;
  const int64_t ld = round8(lk);
  if (segments < 0 || segments >= (int64_t(1) << 31) || slab_rows < 1 ||
      ld > KAT_BIAS_SLAB_CELLS || slab_rows * ld > KAT_BIAS_SLAB_CELLS ||
      slabs != (lq + slab_rows - 1) / slab_rows || slabs >= (int64_t(1) << 31))
    return KAT_ERR_BAD_SHAPE;
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < kat_index_bias_bwd_workspace_bytes(heads, segments))
    return KAT_ERR_WORKSPACE;
  IndexBwd a{};
  a.dout = dout;
  a.sh = dout_stride[0];
  a.si = dout_stride[1];
  a.sj = dout_stride[2];
  a.lq = lq;
  a.lk = lk;
  a.pitch = dout_stride[1] == ld ? ld : lk;
  a.cells = a.pitch == ld ? padded_cells : cells;
  a.seg_begin = seg_begin;
  a.slab_begin = slab_begin;
  a.seg_place = seg_place;
  a.segments = segments;
  a.slab_rows = slab_rows;
  a.heads = heads;
  a.part = static_cast<float*>(workspace);
  int rc = KAT_OK;
  switch (dout_dtype) {
    case KAT_DTYPE_F32: rc = launch_index_bwd<float>(a, slabs, st); break;
    case KAT_DTYPE_F16: rc = launch_index_bwd<__half>(a, slabs, st); break;
    default: rc = launch_index_bwd<__nv_bfloat16>(a, slabs, st); break;
  }
  if (rc) return rc;
  const int64_t sums = int64_t(num_buckets) * heads;
  kat_index_bias_bucket_kernel<<<uint32_t((sums + 31) / 32), 256, 0, st>>>(
      a.part, segments, bucket_begin, num_buckets, heads, d_table, table_dtype);
  return launched();
}

}  // extern "C"
