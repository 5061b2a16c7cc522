// kat_position_bias.cu — learned relative position bias by buckets, forward and backward (C ABI:
// include/kat_position_bias.h).
//
// Distance form.  The bias is constant along diagonals.  Forward: a block looks its diagonals'
// values up once into shared memory; a thread owns 8 columns and walks down the rows, where its
// window of 8 values moves by one: one shared-memory read and a shift for every 16-byte
// store.  Backward: a thread owns 15 neighbouring diagonals and keeps their sums in registers: it
// reads 8 x 8 cells at a time, stepping 8 rows down and 8 columns right, so that every cell is
// read once, in 16-byte accesses, and no two threads add to one sum.
//
// Index form.  Forward: the table's column of a head in shared memory, 8 cells of the index read
// once for several heads.  Backward: a slab of whole rows goes to shared memory in 16-byte
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

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  switch (dtype) {
    case KAT_DTYPE_F32: return static_cast<const float*>(p)[i];
    case KAT_DTYPE_F16: return __half2float(static_cast<const __half*>(p)[i]);
    default: return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
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

// 8 neighbouring values of a row as words; `keep` of them count, the others become zero.
template <typename T> struct Window {
  static constexpr int kWords = 2 * int(sizeof(T));
  uint32_t w[kWords];
};

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
  const int64_t j0 = int64_t(blockIdx.x % a.col_blocks) * a.tx * 8;
  const int64_t i0 = int64_t(blockIdx.x / a.col_blocks) * a.ty * a.rows;
  const int span = a.ty * a.rows;
  const int64_t first = j0 - (i0 + span - 1) - a.offset;   // distance of f[0]
  for (int k = threadIdx.x; k < 8 * a.tx + span - 1; k += kFwdThreads) {
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
  const int64_t j = j0 + 8 * tx;
  const int64_t i = i0 + int64_t(ty) * a.rows;
  if (j >= a.ld || i >= a.lq) return;
  // columns behind lk are zero
  uint32_t keep[Window<T>::kWords];
#pragma unroll
  for (int k = 0; k < Window<T>::kWords; ++k) {
    if constexpr (sizeof(T) == 4) {
      keep[k] = j + k < a.lk ? 0xffffffffu : 0u;
    } else {
      keep[k] = (j + 2 * k < a.lk ? 0xffffu : 0u) | (j + 2 * k + 1 < a.lk ? 0xffff0000u : 0u);
    }
  }
  const U* at = f + 8 * tx + span - 1 - ty * a.rows;   // (i, j)
  Window<T> v;
#pragma unroll
  for (int k = 0; k < Window<T>::kWords; ++k) {
    if constexpr (sizeof(T) == 4) v.w[k] = at[k];
    else v.w[k] = uint32_t(at[2 * k]) | (uint32_t(at[2 * k + 1]) << 16);
  }
  uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t(h) * a.lq + i) * a.ld + j);
  const int64_t step = a.ld * int64_t(sizeof(T)) / 16;
  const int rows = int(a.lq - i < a.rows ? a.lq - i : a.rows);
  for (int r = 0; r < rows; ++r) {
#pragma unroll
    for (int q = 0; q < Window<T>::kWords / 4; ++q)
      out[q] = make_uint4(v.w[4 * q] & keep[4 * q], v.w[4 * q + 1] & keep[4 * q + 1],
                          v.w[4 * q + 2] & keep[4 * q + 2], v.w[4 * q + 3] & keep[4 * q + 3]);
    out += step;
    if (r + 1 == rows) break;
    // one row down: every value moves one column right
    const uint32_t next = *--at;
#pragma unroll
    for (int k = Window<T>::kWords - 1; k > 0; --k) {
      if constexpr (sizeof(T) == 4) v.w[k] = v.w[k - 1];
      else v.w[k] = __funnelshift_l(v.w[k - 1], v.w[k], 16);
    }
    if constexpr (sizeof(T) == 4) v.w[0] = next;
    else v.w[0] = (v.w[0] << 16) | next;
  }
}

// ---------------------------------------------------------------------------
// Distance form, backward.
// ---------------------------------------------------------------------------

constexpr int kBwdThreads = 128;
constexpr int kWin = 16;   // 15 diagonals of a thread, padded

struct DistanceBwd {
  const void* dout;
  int64_t sh, si, sj;
  int64_t lq, lk, offset;
  int32_t causal, groups;    // groups of 8 rows in a split
  int64_t splits, chunks;    // splits of the rows; threads (windows) of a split
  float* part;               // [head][split][chunk][16]
  double* diag;              // [head][lq + lk - 1]
};

template <typename T> __device__ __forceinline__ float load_one(const T* p);
template <> __device__ __forceinline__ float load_one<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float load_one<__half>(const __half* p) {
  return __half2float(*p);
}
template <> __device__ __forceinline__ float load_one<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

// Up to 8 x 8 cells one by one; the loads of one row at a time, so that their addresses do not
// fill the registers.
template <typename T>
__device__ __forceinline__ void add_cells(const T* p, int64_t si, int64_t sj, int rows, int cols,
                                          float (&acc)[15]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (r < rows) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < cols) acc[e - r + 7] += load_one(p + e * sj);
    }
    p += si;
    asm volatile("" ::: "memory");
  }
}

// Where the rows of a gradient start on 16 bytes, `kVec`.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kBwdThreads)
kat_distance_bias_bwd_kernel(const __grid_constant__ DistanceBwd a) {
  const int64_t k = int64_t(blockIdx.x) * kBwdThreads + threadIdx.x;
  if (k >= a.chunks) return;
  const int64_t split = blockIdx.y, h = blockIdx.z;
  const int64_t g0 = split * a.groups;
  const int64_t rows8 = (a.lq + 7) / 8, cols8 = (a.lk + 7) / 8;
  const int64_t g1 = g0 + a.groups < rows8 ? g0 + a.groups : rows8;
  const int64_t c = k - (g0 + a.groups - 1);        // window: diagonals 8c - 7 .. 8c + 7
  if (a.causal && 8 * c - 7 > a.offset) return;     // masked, and never read
  float acc[15];
#pragma unroll
  for (int i = 0; i < 15; ++i) acc[i] = 0.0f;
  const T* base = static_cast<const T*>(a.dout) + h * a.sh;
  const int64_t gb = g0 > -c ? g0 : -c, ge = g1 < cols8 - c ? g1 : cols8 - c;
  for (int64_t g = gb; g < ge; ++g) {
    const int64_t i = 8 * g, j = 8 * (c + g);
    const T* p = base + i * a.si + j * a.sj;
    bool whole = false;
    if constexpr (kVec) {
      whole = i + 8 <= a.lq && j + 8 <= a.lk;
      if (whole) {
        constexpr int kPer = 16 / int(sizeof(T));
        uint4 raw[8][8 / kPer];
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int q = 0; q < 8 / kPer; ++q) raw[r][q] = load_raw<T, kPer>(p + r * a.si + q * kPer);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
#pragma unroll
          for (int q = 0; q < 8 / kPer; ++q) {
            const uint32_t w[4] = {raw[r][q].x, raw[r][q].y, raw[r][q].z, raw[r][q].w};
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
      }
    }
    if (!whole) {
      const int64_t rows = a.lq - i, cols = a.lk - j;
      add_cells<T>(p, a.si, a.sj, int(rows < 8 ? rows : 8), int(cols < 8 ? cols : 8), acc);
    }
  }
  float4* to = reinterpret_cast<float4*>(a.part + ((h * a.splits + split) * a.chunks + k) * kWin);
  to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  to[2] = make_float4(acc[8], acc[9], acc[10], acc[11]);
  to[3] = make_float4(acc[12], acc[13], acc[14], 0.0f);
}

// One sum for each diagonal: two windows hold it in every split.
__global__ void __launch_bounds__(256)
kat_distance_bias_diag_kernel(const __grid_constant__ DistanceBwd a) {
  const int64_t count = a.lq + a.lk - 1;
  const int64_t k = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (k >= count) return;
  const int64_t h = blockIdx.y;
  const int64_t d = k - (a.lq - 1);
  double sum = 0.0;
  if (!a.causal || d <= a.offset) {
    const int64_t c = d >= 0 ? d / 8 : -((7 - d) / 8);
    const int o = int(d - 8 * c);
    for (int64_t s = 0; s < a.splits; ++s) {
      const int64_t at = c + s * a.groups + a.groups - 1;
      const float* part = a.part + ((h * a.splits + s) * a.chunks + at) * kWin;
      if (at >= 0 && at < a.chunks) sum += double(part[o + 7]);
      if (o > 0 && at + 1 >= 0 && at + 1 < a.chunks) sum += double(part[kWin + o - 1]);
    }
  }
  a.diag[h * count + k] = sum;
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
constexpr int kIdxSmem = 64 * 1024;       // table columns of a block
constexpr int kIdxSmemMost = 200 * 1024;  // above this even one column stays in global memory

struct IndexFwd {
  const void* table;
  const int32_t* index;
  void* out;
  int64_t chunks;          // lq * ld / 8
  int32_t table_dtype, num_buckets, heads;
  int32_t group;           // heads of a block
};

// Neighbouring cells of a grid's row have neighbouring buckets, 8 apart from lane to lane: one word
// more every 32 keeps them in different banks.
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
    for (int64_t k = threadIdx.x; k < int64_t(a.num_buckets + 1) * heads; k += kIdxThreads) {
      const int b = int(k / heads), h = int(k % heads);
      f[h * pitch + spread(b)] =
          b == a.num_buckets ? U(0)
                             : bits_of<T>(load_any(a.table, a.table_dtype,
                                                   int64_t(b) * a.heads + h0 + h));
    }
    __syncthreads();
  }
  for (int64_t k = int64_t(blockIdx.x) * kIdxThreads + threadIdx.x; k < a.chunks;
       k += int64_t(gridDim.x) * kIdxThreads) {
    const int4 lo = __ldg(reinterpret_cast<const int4*>(a.index) + 2 * k);
    const int4 hi = __ldg(reinterpret_cast<const int4*>(a.index) + 2 * k + 1);
    const int b[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    int at[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) at[e] = kSmem ? spread(b[e]) : b[e];
    for (int h = 0; h < heads; ++h) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (kSmem) {
          v[e] = f[h * pitch + at[e]];
        } else {
          v[e] = at[e] == a.num_buckets
                     ? 0u
                     : uint32_t(bits_of<T>(load_any(a.table, a.table_dtype,
                                                    int64_t(at[e]) * a.heads + h0 + h)));
        }
      }
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) +
                                            (int64_t(h0 + h) * a.chunks + k) * 8);
      if constexpr (sizeof(T) == 4) {
        out[0] = make_uint4(v[0], v[1], v[2], v[3]);
        out[1] = make_uint4(v[4], v[5], v[6], v[7]);
      } else {
        out[0] = make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16),
                            v[6] | (v[7] << 16));
      }
    }
  }
}

struct IndexBwd {
  const void* dout;
  int64_t sh, si, sj;
  int64_t lq, lk, ld;
  const uint16_t* cells;
  const int32_t* seg_begin;
  const int32_t* slab_begin;
  int64_t segments;
  int32_t slab_rows;
  float* part;             // [head][segment]
};

template <typename T, bool kVec>
__global__ void __launch_bounds__(kIdxThreads)
kat_index_bias_bwd_kernel(const __grid_constant__ IndexBwd a) {
  extern __shared__ uint4 slab_smem[];
  T* s = reinterpret_cast<T*>(slab_smem);
  const int64_t h = blockIdx.y;
  const int64_t i0 = int64_t(blockIdx.x) * a.slab_rows;
  const int rows = int(a.lq - i0 < a.slab_rows ? a.lq - i0 : a.slab_rows);
  const T* base = static_cast<const T*>(a.dout) + h * a.sh + i0 * a.si;
  const uint32_t ld = uint32_t(a.ld);
  if constexpr (kVec) {
    constexpr int kPer = 16 / int(sizeof(T));
    const uint32_t per_row = ld / kPer, full = uint32_t(a.lk) / kPer;
    for (uint32_t k = threadIdx.x; k < uint32_t(rows) * per_row; k += kIdxThreads) {
      const uint32_t r = k / per_row, q = k % per_row;
      const T* p = base + int64_t(r) * a.si + q * kPer;
      if (q < full) {
        slab_smem[k] = load_raw<T, kPer>(p);
      } else {
        for (uint32_t e = 0; e < kPer && q * kPer + e < uint32_t(a.lk); ++e)
          s[k * kPer + e] = p[e];
      }
    }
  } else {
    for (uint32_t k = threadIdx.x; k < uint32_t(rows) * ld; k += kIdxThreads) {
      const uint32_t r = k / ld, j = k % ld;
      if (j < uint32_t(a.lk)) s[k] = base[int64_t(r) * a.si + int64_t(j) * a.sj];
    }
  }
  __syncthreads();
  const int32_t end = __ldg(a.slab_begin + blockIdx.x + 1);
  for (int32_t g = __ldg(a.slab_begin + blockIdx.x) + int(threadIdx.x); g < end; g += kIdxThreads) {
    float sum = 0.0f;
    const int32_t last = __ldg(a.seg_begin + g + 1);
    for (int32_t k = __ldg(a.seg_begin + g); k < last; ++k) {
      if constexpr (sizeof(T) == 4) sum += s[__ldg(a.cells + k)];
      else sum += Codec<T>::unpack1(reinterpret_cast<const uint16_t*>(s)[__ldg(a.cells + k)]);
    }
    a.part[h * a.segments + g] = sum;
  }
}

// The segments of a bucket for one head, by 8 lanes.
__global__ void __launch_bounds__(256)
kat_index_bias_bucket_kernel(const float* __restrict__ part, int64_t segments,
                             const int32_t* __restrict__ by_bucket,
                             const int32_t* __restrict__ bucket_begin, int num_buckets, int heads,
                             void* d_table, int table_dtype) {
  const int64_t k = int64_t(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const int lane = threadIdx.x & 7;
  const bool live = k < int64_t(num_buckets) * heads;
  const int b = live ? int(k % num_buckets) : 0, h = live ? int(k / num_buckets) : 0;
  double sum = 0.0;
  if (live) {
    const int32_t end = bucket_begin[b + 1];
    for (int32_t g = bucket_begin[b] + lane; g < end; g += 8)
      sum += double(part[int64_t(h) * segments + by_bucket[g]]);
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
// Rows of a split: as many as leave enough windows for the whole device (148 SMs x 1024 threads),
// since every window of a split costs 64 bytes of partial sums for 128 bytes a group.
DistancePlan distance_plan(int32_t heads, int64_t lq, int64_t lk) {
  const int64_t rows8 = (lq + 7) / 8, cols8 = (lk + 7) / 8;
  int64_t g = 32;
  auto splits = [&](int64_t n) { return (rows8 + n - 1) / n; };
  while (g > 1 && heads * splits(g) * (cols8 + g - 1) < 148 * 1024) g /= 2;
  while (splits(g) > 65535) g *= 2;
  DistancePlan p;
  p.groups = int32_t(g);
  p.splits = splits(g);
  p.chunks = cols8 + g - 1;
  p.part = size_t(heads) * size_t(p.splits) * size_t(p.chunks) * kWin * sizeof(float);
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
void launch_distance_bwd(const DistanceBwd& a, bool vec, dim3 grid, cudaStream_t st) {
  if (vec) kat_distance_bias_bwd_kernel<T, true><<<grid, kBwdThreads, 0, st>>>(a);
  else kat_distance_bias_bwd_kernel<T, false><<<grid, kBwdThreads, 0, st>>>(a);
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
  // large ones: a block takes several runs of cells, so that it loads its table columns once
  const int64_t most = (148 * 6 + head_blocks - 1) / head_blocks;
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

template <typename T, bool kVec>
int launch_index_bwd_v(const IndexBwd& a, dim3 grid, cudaStream_t st) {
  const size_t bytes = size_t(a.slab_rows) * size_t(a.ld) * sizeof(T);
  if (int rc = set_smem(kat_index_bias_bwd_kernel<T, kVec>, bytes)) return rc;
  kat_index_bias_bwd_kernel<T, kVec><<<grid, kIdxThreads, bytes, st>>>(a);
  return launched();
}
template <typename T>
int launch_index_bwd(const IndexBwd& a, bool vec, dim3 grid, cudaStream_t st) {
  return vec ? launch_index_bwd_v<T, true>(a, grid, st) : launch_index_bwd_v<T, false>(a, grid, st);
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
  const int64_t chunks = a.ld / 8;
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
      (size_t(8 * a.tx + a.ty * a.rows - 1) * elem_size(out_dtype) + 3) / 4 * 4;
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
  return distance_plan(heads, lq, lk).total;
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
  const DistancePlan plan = distance_plan(heads, lq, lk);
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
  a.part = static_cast<float*>(workspace);
  a.diag = reinterpret_cast<double*>(static_cast<uint8_t*>(workspace) + plan.part);
  const dim3 grid{uint32_t((plan.chunks + kBwdThreads - 1) / kBwdThreads), uint32_t(plan.splits),
                  uint32_t(heads)};
  const bool vec = vector_rows(dout, dout_dtype, dout_stride);
  switch (dout_dtype) {
    case KAT_DTYPE_F32: launch_distance_bwd<float>(a, vec, grid, st); break;
    case KAT_DTYPE_F16: launch_distance_bwd<__half>(a, vec, grid, st); break;
    default: launch_distance_bwd<__nv_bfloat16>(a, vec, grid, st); break;
  }
  if (int rc = launched()) return rc;
  kat_distance_bias_diag_kernel<<<dim3(uint32_t((lq + lk - 1 + 255) / 256), uint32_t(heads)), 256,
                                  0, st>>>(a);
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
  a.chunks = lq * (round8(lk) / 8);
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
                       const uint16_t* cells, const int32_t* seg_begin, int64_t segments,
                       const int32_t* slab_begin, int64_t slabs, int32_t slab_rows,
                       const int32_t* by_bucket, const int32_t* bucket_begin, void* d_table,
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
  if (dout == nullptr || dout_stride == nullptr || cells == nullptr || seg_begin == nullptr ||
      slab_begin == nullptr || by_bucket == nullptr || bucket_begin == nullptr)
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
  a.ld = ld;
  a.cells = cells;
  a.seg_begin = seg_begin;
  a.slab_begin = slab_begin;
  a.segments = segments;
  a.slab_rows = slab_rows;
  a.part = static_cast<float*>(workspace);
  const dim3 grid{uint32_t(slabs), uint32_t(heads)};
  const bool vec = vector_rows(dout, dout_dtype, dout_stride);
  int rc = KAT_OK;
  switch (dout_dtype) {
    case KAT_DTYPE_F32: rc = launch_index_bwd<float>(a, vec, grid, st); break;
    case KAT_DTYPE_F16: rc = launch_index_bwd<__half>(a, vec, grid, st); break;
    default: rc = launch_index_bwd<__nv_bfloat16>(a, vec, grid, st); break;
  }
  if (rc) return rc;
  const int64_t sums = int64_t(num_buckets) * heads;
  kat_index_bias_bucket_kernel<<<uint32_t((sums + 31) / 32), 256, 0, st>>>(
      a.part, segments, by_bucket, bucket_begin, num_buckets, heads, d_table, table_dtype);
  return launched();
}

}  // extern "C"
