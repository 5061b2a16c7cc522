// kat_qk_norm_rope.cu — norm of queries and keys for each head with the position rotation, in one
// pass, forward and backward (C ABI: include/kat_qk_norm_rope.h).
//
// A head's vector is read once, kept in registers as fp32, and written once.  In the vector
// kernels a group of LANES lanes holds a head, 16 values to a lane in two chunks of 8 chosen so
// that both values of a pair lie in the same lane (chunks rot/2 apart for pairs (i, i + rot/2)),
// so the rotation needs no exchange and every access is a 16-byte one.  The sums over a head are
// shuffles inside the group.  A group takes runs of up to four consecutive heads (heads are numbered
// through all tokens, a token's heads next to each other), so that a token's angles are mostly
// loaded once a run, and walks the runs with a grid stride.
// What bounds it is HBM; what it takes is enough bytes in flight.  Loads into registers alone kept
// too few (x[128,197,12+12,64] bf16: forward 37 us, backward 76 us, 64 and 62 % of the copy rate):
// each thread copies the values of its next heads with cp.async into slots of its own in
// shared memory, three heads ahead, which needs no barrier, only its own wait: 31.8 and 54.4 us, and
// 4.3 us for the weights' sums (x[2,8191,32+8,128] bf16: 61, 89 and 4.4 us).
// Any other size, stride or alignment takes the general kernels, one warp to a head.

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <mutex>

#include "kat_rational.h"
#include "kat_qk_norm_rope.h"

namespace {

#include "kat_math.cuh"

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxHeadDim = 1024;
constexpr int kVecMaxHeadDim = 256;
constexpr int kChunk = 8;
constexpr int kFwdBlocksPerSm = 3;
constexpr int kBwdBlocksPerSm = 2;   // also the partial rows of the weights' gradients per SM
constexpr int kMaxRun = 4;           // heads a group takes in a row

// Division of n < 2^31 by an invariant d >= 1: with l = ceil(log2 d) and
// m = floor(2^(31 + l) / d) + 1 (below 2^32), n / d = (n m) >> (31 + l).
struct Divider {
  uint32_t d, m, shift;
};

struct Stream {
  const void* x;
  const void* dy;
  void* out;
  const void* weight;
  float* dweight;
  int64_t xs[3], ds[3], os[3];
  Divider heads;
  uint32_t rows;       // heads of all tokens
  uint32_t run;        // consecutive heads of a group's turn
};

struct Params {
  Stream s[KAT_MAX_HEAD_STREAMS];
  Divider tokens;
  int32_t head_dim, rot_dim, weight_dtype;
  float eps, inv_dim;
  const float* cos_table;
  const float* sin_table;
  int64_t table_rows;
  const int64_t* positions;
  int64_t ps[2];
  float* partial;      // backward: [stream][block][head_dim]
};

__device__ __forceinline__ void divide(uint32_t n, const Divider& v, uint32_t& q, uint32_t& r) {
  q = uint32_t((uint64_t(n) * v.m) >> v.shift);
  r = n - q * v.d;
}

// One head of one token: its place and its table row.
struct Where {
  uint32_t b, t, h, token;
};
__device__ __forceinline__ Where locate(const Params& p, const Stream& s, uint32_t row) {
  Where w;
  divide(row, s.heads, w.token, w.h);
  divide(w.token, p.tokens, w.b, w.t);
  return w;
}
struct Row {
  int64_t pos;
  bool in_table;
};
__device__ __forceinline__ Row table_row(const Params& p, const Where& w) {
  Row r;
  r.pos = p.positions != nullptr
              ? __ldg(p.positions + int64_t(w.b) * p.ps[0] + int64_t(w.t) * p.ps[1])
              : int64_t(w.t);
  r.in_table = p.rot_dim == 0 || (r.pos >= 0 && r.pos < p.table_rows);
  return r;
}
__device__ __forceinline__ int64_t offset(const int64_t (&st)[3], const Where& w) {
  return int64_t(w.b) * st[0] + int64_t(w.t) * st[1] + int64_t(w.h) * st[2];
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int i) {
  switch (dtype) {
    case KAT_DTYPE_F32: return __ldg(static_cast<const float*>(p) + i);
    case KAT_DTYPE_F16: return __half2float(__ldg(static_cast<const __half*>(p) + i));
    default: return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
  }
}

// ---------------------------------------------------------------------------
// Vector kernels.
// ---------------------------------------------------------------------------

// Chunks of 8 values as they lie in memory.
template <typename T> struct Raw {
  static constexpr int kWords = kChunk * int(sizeof(T)) / 16;
  uint4 w[kWords];
};
template <typename T> __device__ __forceinline__ Raw<T> load8(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = load_raw<T, 16 / int(sizeof(T))>(p + i * (16 / int(sizeof(T))));
  return r;
}
template <typename T> __device__ __forceinline__ Raw<T> zero8() {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = make_uint4(0u, 0u, 0u, 0u);
  return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
template <typename T> __device__ __forceinline__ void to_float(const Raw<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i + 0] = __uint_as_float(r.w[i].x);
      f[4 * i + 1] = __uint_as_float(r.w[i].y);
      f[4 * i + 2] = __uint_as_float(r.w[i].z);
      f[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = Codec<T>::unpack_word(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T> __device__ __forceinline__ Raw<T> from_float(const float (&f)[8]) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.w[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]),
                          __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Codec<T>::pack_word(make_float2(f[2 * i], f[2 * i + 1]));
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

// What lane l of a group holds: values a .. a + 7 and b .. b + 7, with the angles of their pairs.
// Pairs (i, i + rot/2): lanes below rot/16 hold chunks rot/2 apart (8 angles from ca on), the
// others two chunks behind rot.  Pairs (2i, 2i + 1): chunks D/2 apart, each with 4 angles
// of its own (from ca and cb on) if it lies below rot.
struct Part {
  int a, b, ca, cb;
  bool turn_a, turn_b, active;
};
template <bool INTER>
__device__ __forceinline__ Part part_of(int l, int dim, int rot) {
  Part p;
  p.active = 16 * l < dim;
  if constexpr (INTER) {
    p.a = 8 * l;
    p.b = dim / 2 + 8 * l;
    p.ca = p.a / 2;
    p.cb = p.b / 2;
    p.turn_a = p.active && p.a < rot;
    p.turn_b = p.active && p.b < rot;
  } else {
    p.turn_a = p.turn_b = 16 * l < rot;
    p.a = p.turn_a ? 8 * l : 16 * l;
    p.b = p.turn_a ? rot / 2 + 8 * l : 16 * l + 8;
    p.ca = 8 * l;
    p.cb = 8 * l + 4;
  }
  return p;
}

struct Angles {
  float c[8], s[8];   // [0..3] at ca, [4..7] at cb
};
__device__ __forceinline__ void load4(const float* p, float* f) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
__device__ __forceinline__ Angles load_angles(const Params& p, const Part& part, const Row& w) {
  Angles g;
#pragma unroll
  for (int i = 0; i < 8; ++i) { g.c[i] = 1.0f; g.s[i] = 0.0f; }
  if (w.in_table) {
    const int64_t row = w.pos * (p.rot_dim / 2);
    if (part.turn_a) {
      load4(p.cos_table + row + part.ca, g.c);
      load4(p.sin_table + row + part.ca, g.s);
    }
    if (part.turn_b) {
      load4(p.cos_table + row + part.cb, g.c + 4);
      load4(p.sin_table + row + part.cb, g.s + 4);
    }
  }
  return g;
}
// Turns the pairs by the angles, or back by them.
template <bool INTER, bool BACK>
__device__ __forceinline__ void turn_pairs(float (&a)[8], float (&b)[8], const Angles& g) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sa = BACK ? -g.s[i] : g.s[i], sb = BACK ? -g.s[4 + i] : g.s[4 + i];
      const float x = a[2 * i], y = a[2 * i + 1], u = b[2 * i], v = b[2 * i + 1];
      a[2 * i] = x * g.c[i] - y * sa;
      a[2 * i + 1] = x * sa + y * g.c[i];
      b[2 * i] = u * g.c[4 + i] - v * sb;
      b[2 * i + 1] = u * sb + v * g.c[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = BACK ? -g.s[i] : g.s[i];
      const float x = a[i], y = b[i];
      a[i] = x * g.c[i] - y * s;
      b[i] = x * s + y * g.c[i];
    }
  }
}

template <int LANES> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int k = LANES / 2; k > 0; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
  return v;
}
__device__ __forceinline__ float norm_of(const Params& p, bool in_table, float sum) {
  const float r = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
  return in_table ? r : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ void load_weights(const Params& p, const Stream& s, const Part& part,
                                             float (&wa)[8], float (&wb)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool any = s.weight != nullptr && part.active;
    wa[i] = any ? load_any(s.weight, p.weight_dtype, part.a + i) : 1.0f;
    wb[i] = any ? load_any(s.weight, p.weight_dtype, part.b + i) : 1.0f;
  }
}

// A thread's ring of slots in shared memory: kChunks pieces of 8 values to a stage, three stages
// ahead (two of fp32, whose stages are twice as large).
template <typename T, int kChunks> struct Ring {
  static constexpr int kStages = sizeof(T) == 4 ? 3 : 4;
  static constexpr int kWords = Raw<T>::kWords;
  static constexpr uint32_t kBytes = uint32_t(kStages) * kChunks * kWords * kThreads * 16;
  uint32_t base;   // shared address of this thread's first slot
  __device__ __forceinline__ explicit Ring(const void* smem)
      : base(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16u) {}
  __device__ __forceinline__ uint32_t slot(int stage, int chunk, int word) const {
    return base + uint32_t(((stage * kChunks + chunk) * kWords + word) * kThreads * 16);
  }
  __device__ __forceinline__ void copy(int stage, int chunk, const T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(
                       slot(stage, chunk, i)), "l"(p + i * (16 / int(sizeof(T)))) : "memory");
  }
  __device__ __forceinline__ Raw<T> read(int stage, int chunk) const {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.w[i].x), "=r"(r.w[i].y), "=r"(r.w[i].z), "=r"(r.w[i].w)
                   : "r"(slot(stage, chunk, i)) : "memory");
    return r;
  }
  __device__ __forceinline__ static void commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // all but the newest kStages - 2 groups of copies of this thread have landed
  __device__ __forceinline__ static void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
  }
};

// The heads of a group of lanes, one after the other: turn k takes head k % run of the group's
// run k / run.  Every lane of a warp makes the same number of turns (the shuffles need them
// all); turns behind the last head are idle.
template <int LANES> struct Walk {
  uint32_t group, stride, run, rows, turns;
  uint32_t at, k;     // the run and the place in it of the next turn
  __device__ __forceinline__ Walk(const Stream& s) {
    constexpr uint32_t kPerWarp = 32 / LANES;
    const uint32_t warp = (blockIdx.x * kThreads + threadIdx.x) / 32;
    run = s.run;
    rows = s.rows;
    group = warp * kPerWarp + (threadIdx.x & 31) / LANES;
    stride = gridDim.x * (kThreads / LANES);
    const uint32_t runs = (rows + run - 1) / run, first = warp * kPerWarp;
    turns = first < runs ? ((runs - first + stride - 1) / stride) * run : 0;
    at = group;
    k = 0;
  }
  // the next turn's head (past the end: >= rows)
  __device__ __forceinline__ uint32_t next() {
    const uint64_t row = uint64_t(at) * run + k;
    if (++k == run) {
      k = 0;
      at += stride;
    }
    return row < rows ? uint32_t(row) : 0xffffffffu;
  }
};

template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads, kFwdBlocksPerSm)
kat_head_fwd_kernel(const __grid_constant__ Params p) {
  using R = Ring<T, 2>;
  extern __shared__ uint4 ring_smem[];
  const R ring(ring_smem);
  const Stream& s = p.s[blockIdx.y];
  const Part part = part_of<INTER>(threadIdx.x % LANES, p.head_dim, p.rot_dim);
  const T* x = static_cast<const T*>(s.x);
  T* out = static_cast<T*>(s.out);
  float wa[8], wb[8];
  load_weights(p, s, part, wa, wb);
  Walk<LANES> ahead(s), now(s);
  auto fetch = [&](int stage) {
    const uint32_t row = ahead.next();
    if (row != 0xffffffffu && part.active) {
      const T* from = x + offset(s.xs, locate(p, s, row));
      ring.copy(stage, 0, from + part.a);
      ring.copy(stage, 1, from + part.b);
    }
    R::commit();
  };
#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) fetch(i);
  uint32_t token = 0xffffffffu;
  bool in_table = true;
  Angles g;
  int stage = 0;
  for (uint32_t turn = 0; turn < now.turns; ++turn) {
    const uint32_t row = now.next();
    const bool live = row != 0xffffffffu && part.active;
    const Where w = locate(p, s, row != 0xffffffffu ? row : 0u);
    if (w.token != token) {
      const Row tr = table_row(p, w);
      g = load_angles(p, part, tr);
      in_table = tr.in_table;
      token = w.token;
    }
    R::wait();
    const Raw<T> ra = live ? ring.read(stage, 0) : zero8<T>();
    const Raw<T> rb = live ? ring.read(stage, 1) : zero8<T>();
    fetch(stage == 0 ? R::kStages - 1 : stage - 1);
    if (++stage == R::kStages) stage = 0;
    float a[8], b[8];
    to_float<T>(ra, a);
    to_float<T>(rb, b);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
    const float r = norm_of(p, in_table, group_sum<LANES>(sum));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = a[i] * r * wa[i];
      b[i] = b[i] * r * wb[i];
    }
    turn_pairs<INTER, false>(a, b, g);
    if (live) {
      T* to = out + offset(s.os, w);
      store8(to + part.a, from_float<T>(a));
      store8(to + part.b, from_float<T>(b));
    }
  }
}

template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads, kBwdBlocksPerSm)
kat_head_bwd_kernel(const __grid_constant__ Params p) {
  using R = Ring<T, 4>;
  extern __shared__ uint4 ring_smem[];
  const R ring(ring_smem);
  const Stream& s = p.s[blockIdx.y];
  const Part part = part_of<INTER>(threadIdx.x % LANES, p.head_dim, p.rot_dim);
  const T* x = static_cast<const T*>(s.x);
  const T* dy = static_cast<const T*>(s.dy);
  T* out = static_cast<T*>(s.out);
  const bool copy = x == nullptr;  // values that passed by: their gradient is copied
  Walk<LANES> ahead(s), now(s);
  auto fetch = [&](int stage) {
    const uint32_t row = ahead.next();
    if (row != 0xffffffffu && part.active) {
      const Where w = locate(p, s, row);
      if (!copy) {
        const T* from = x + offset(s.xs, w);
        ring.copy(stage, 0, from + part.a);
        ring.copy(stage, 1, from + part.b);
      }
      const T* from = dy + offset(s.ds, w);
      ring.copy(stage, 2, from + part.a);
      ring.copy(stage, 3, from + part.b);
    }
    R::commit();
  };
#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) fetch(i);
  int stage = 0;
  if (copy) {
    for (uint32_t turn = 0; turn < now.turns; ++turn) {
      const uint32_t row = now.next();
      R::wait();
      if (row != 0xffffffffu && part.active) {
        T* to = out + offset(s.os, locate(p, s, row));
        store8(to + part.a, ring.read(stage, 2));
        store8(to + part.b, ring.read(stage, 3));
      }
      fetch(stage == 0 ? R::kStages - 1 : stage - 1);
      if (++stage == R::kStages) stage = 0;
    }
    return;
  }
  float wa[8], wb[8], da[8], db[8];
  load_weights(p, s, part, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.0f;
  uint32_t token = 0xffffffffu;
  bool in_table = true;
  Angles g;
  for (uint32_t turn = 0; turn < now.turns; ++turn) {
    const uint32_t row = now.next();
    const bool live = row != 0xffffffffu && part.active;
    const Where w = locate(p, s, row != 0xffffffffu ? row : 0u);
    if (w.token != token) {
      const Row tr = table_row(p, w);
      g = load_angles(p, part, tr);
      in_table = tr.in_table;
      token = w.token;
    }
    R::wait();
    const Raw<T> ra = live ? ring.read(stage, 0) : zero8<T>();
    const Raw<T> rb = live ? ring.read(stage, 1) : zero8<T>();
    const Raw<T> rga = live ? ring.read(stage, 2) : zero8<T>();
    const Raw<T> rgb = live ? ring.read(stage, 3) : zero8<T>();
    fetch(stage == 0 ? R::kStages - 1 : stage - 1);
    if (++stage == R::kStages) stage = 0;
    float a[8], b[8], ga[8], gb[8];
    to_float<T>(ra, a);
    to_float<T>(rb, b);
    to_float<T>(rga, ga);
    to_float<T>(rgb, gb);
    turn_pairs<INTER, true>(ga, gb, g);
    float sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
      dot = fmaf(ga[i] * wa[i], a[i], fmaf(gb[i] * wb[i], b[i], dot));
    }
    sum = group_sum<LANES>(sum);
    dot = group_sum<LANES>(dot);
    const float r = norm_of(p, in_table, sum);
    const float mean = dot * r * p.inv_dim;   // mean(dn w x r)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ha = a[i] * r, hb = b[i] * r;
      a[i] = r * (ga[i] * wa[i] - ha * mean);
      b[i] = r * (gb[i] * wb[i] - hb * mean);
      if (live) {
        da[i] = fmaf(ga[i], ha, da[i]);
        db[i] = fmaf(gb[i], hb, db[i]);
      }
    }
    if (live) {
      T* to = out + offset(s.os, w);
      store8(to + part.a, from_float<T>(a));
      store8(to + part.b, from_float<T>(b));
    }
  }
  if (s.dweight == nullptr) return;
  // groups of a warp, then the warps, in a fixed order
  __shared__ float acc[kWarps][kVecMaxHeadDim];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int k = 16; k >= LANES; k >>= 1) {
      da[i] += __shfl_xor_sync(0xffffffffu, da[i], k);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], k);
    }
  }
  if ((threadIdx.x & 31) < LANES && part.active) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[threadIdx.x >> 5][part.a + i] = da[i];
      acc[threadIdx.x >> 5][part.b + i] = db[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < p.head_dim) {
    float sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) sum += acc[w][threadIdx.x];
    p.partial[(int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * p.head_dim + threadIdx.x] = sum;
  }
}

// ---------------------------------------------------------------------------
// General kernels: one warp to a head, one value at a time, the partner of a pair read again.
// ---------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float value_of(const T* p);
template <> __device__ __forceinline__ float value_of<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float value_of<__half>(const __half* p) {
  return __half2float(*p);
}
template <> __device__ __forceinline__ float value_of<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) {
  return __float2half_rn(v);
}
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// The partner of value i of a rotated pair, whether i is the first of the two, and the angle.
struct Pair {
  int other, angle;
  bool first;
};
template <bool INTER> __device__ __forceinline__ Pair pair_of(int i, int rot) {
  Pair q;
  if constexpr (INTER) {
    q.other = i ^ 1;
    q.angle = i >> 1;
    q.first = (i & 1) == 0;
  } else {
    q.first = i < rot / 2;
    q.other = q.first ? i + rot / 2 : i - rot / 2;
    q.angle = q.first ? i : i - rot / 2;
  }
  return q;
}
__device__ __forceinline__ float warp_sum(float v) { return group_sum<32>(v); }
__device__ __forceinline__ float weight_of(const Params& p, const Stream& s, int i) {
  return s.weight != nullptr ? load_any(s.weight, p.weight_dtype, i) : 1.0f;
}

template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads)
kat_head_fwd_any_kernel(const __grid_constant__ Params p) {
  const Stream& s = p.s[blockIdx.y];
  const int lane = threadIdx.x & 31;
  for (uint64_t row = uint64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); row < s.rows;
       row += uint64_t(gridDim.x) * kWarps) {
    const Where w = locate(p, s, uint32_t(row));
    const Row tr = table_row(p, w);
    const T* x = static_cast<const T*>(s.x) + offset(s.xs, w);
    T* out = static_cast<T*>(s.out) + offset(s.os, w);
    float sum = 0.0f;
    for (int i = lane; i < p.head_dim; i += 32) {
      const float v = value_of(x + i);
      sum = fmaf(v, v, sum);
    }
    const float r = norm_of(p, tr.in_table, warp_sum(sum));
    const int64_t angles = tr.pos * (p.rot_dim / 2);
    for (int i = lane; i < p.head_dim; i += 32) {
      float y = value_of(x + i) * r * weight_of(p, s, i);
      if (i < p.rot_dim && tr.in_table) {
        const Pair q = pair_of<INTER>(i, p.rot_dim);
        const float z = value_of(x + q.other) * r * weight_of(p, s, q.other);
        const float c = __ldg(p.cos_table + angles + q.angle);
        const float sn = __ldg(p.sin_table + angles + q.angle);
        y = q.first ? y * c - z * sn : z * sn + y * c;
      }
      out[i] = rounded<T>(y);
    }
  }
}

template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads)
kat_head_bwd_any_kernel(const __grid_constant__ Params p) {
  extern __shared__ float any_acc[];  // [warp][head_dim]: lane l owns values l, l + 32, ...
  const Stream& s = p.s[blockIdx.y];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* acc = any_acc + warp * p.head_dim;
  for (int i = lane; i < p.head_dim; i += 32) acc[i] = 0.0f;
  for (uint64_t row = uint64_t(blockIdx.x) * kWarps + warp; row < s.rows;
       row += uint64_t(gridDim.x) * kWarps) {
    const Where w = locate(p, s, uint32_t(row));
    const T* dy = static_cast<const T*>(s.dy) + offset(s.ds, w);
    T* out = static_cast<T*>(s.out) + offset(s.os, w);
    if (s.x == nullptr) {
      for (int i = lane; i < p.head_dim; i += 32) out[i] = dy[i];
      continue;
    }
    const Row tr = table_row(p, w);
    const T* x = static_cast<const T*>(s.x) + offset(s.xs, w);
    const int64_t angles = tr.pos * (p.rot_dim / 2);
    auto back = [&](int i) {
      float g = value_of(dy + i);
      if (i < p.rot_dim && tr.in_table) {
        const Pair q = pair_of<INTER>(i, p.rot_dim);
        const float z = value_of(dy + q.other);
        const float c = __ldg(p.cos_table + angles + q.angle);
        const float sn = __ldg(p.sin_table + angles + q.angle);
        g = q.first ? g * c + z * sn : g * c - z * sn;
      }
      return g;
    };
    float sum = 0.0f, dot = 0.0f;
    for (int i = lane; i < p.head_dim; i += 32) {
      const float v = value_of(x + i);
      sum = fmaf(v, v, sum);
      dot = fmaf(back(i) * weight_of(p, s, i), v, dot);
    }
    sum = warp_sum(sum);
    dot = warp_sum(dot);
    const float r = norm_of(p, tr.in_table, sum);
    const float mean = dot * r * p.inv_dim;
    for (int i = lane; i < p.head_dim; i += 32) {
      const float g = back(i), h = value_of(x + i) * r;
      out[i] = rounded<T>(r * (g * weight_of(p, s, i) - h * mean));
      acc[i] = fmaf(g, h, acc[i]);
    }
  }
  if (s.dweight == nullptr || s.x == nullptr) return;
  __syncthreads();
  for (int i = threadIdx.x; i < p.head_dim; i += kThreads) {
    float sum = 0.0f;
    for (int k = 0; k < kWarps; ++k) sum += any_acc[k * p.head_dim + i];
    p.partial[(int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * p.head_dim + i] = sum;
  }
}

// dweight = the blocks' partial rows added up in fp64: 32 columns to a block, 32 runs of rows (8 runs
// of 74 rows each took 9 us, as long as the loads one after the other).
__global__ void __launch_bounds__(1024)
kat_head_dweight_kernel(const __grid_constant__ Params p, int blocks) {
  const Stream& s = p.s[blockIdx.y];
  if (s.dweight == nullptr || s.x == nullptr) return;
  __shared__ double acc[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + tx;
  double sum = 0.0;
  if (col < p.head_dim) {
    const float* src = p.partial + int64_t(blockIdx.y) * blocks * p.head_dim + col;
#pragma unroll 4
    for (int b = ty; b < blocks; b += 32) sum += double(src[int64_t(b) * p.head_dim]);
  }
  acc[ty][tx] = sum;
  __syncthreads();
  // a warp to a column, its runs in a fixed tree
  sum = acc[tx][ty];
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  const int mine = blockIdx.x * 32 + ty;
  if (tx == 0 && mine < p.head_dim) s.dweight[mine] = float(sum);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

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

Divider divider(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  return {d, uint32_t((uint64_t(1) << (31 + l)) / d + 1), 31 + l};
}

int elem_size(int dtype) { return dtype == KAT_DTYPE_F32 ? 4 : 2; }
bool known(int dtype) {
  return dtype == KAT_DTYPE_F32 || dtype == KAT_DTYPE_F16 || dtype == KAT_DTYPE_BF16;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks the call and fills in `p`; *vec says whether the vector kernels take it, *rows the
// longest stream.
int make_params(const kat_head_problem* q, const kat_head_stream* streams, int32_t count,
                bool backward, Params* p, bool* vec, uint32_t* rows) {
  if (q == nullptr || streams == nullptr) return KAT_ERR_NULL_POINTER;
  if (!known(q->dtype) || !known(q->weight_dtype)) return KAT_ERR_BAD_DTYPE;
  if (count < 1 || count > KAT_MAX_HEAD_STREAMS || q->batch < 0 || q->tokens < 0 ||
      q->head_dim < 1 || q->head_dim > kMaxHeadDim || q->rot_dim < 0 ||
      q->rot_dim > q->head_dim || q->rot_dim % 2 != 0)
    return KAT_ERR_BAD_SHAPE;
  *rows = 0;
  for (int i = 0; i < count; ++i) {
    if (streams[i].heads < 0) return KAT_ERR_BAD_SHAPE;
    const int64_t most = (int64_t(1) << 31) - 1;
    int64_t n = streams[i].heads;
    if (q->tokens != 0 && n > most / q->tokens) return KAT_ERR_BAD_SHAPE;
    n *= q->tokens;
    if (q->batch != 0 && n > most / q->batch) return KAT_ERR_BAD_SHAPE;
    n *= q->batch;
    p->s[i].rows = uint32_t(n);
    if (uint32_t(n) > *rows) *rows = uint32_t(n);
    if (backward && streams[i].x == nullptr && streams[i].dweight != nullptr && n != 0)
      return KAT_ERR_NULL_POINTER;   // a copied stream has no weights
    p->s[i].dweight = streams[i].dweight;
  }
  p->head_dim = q->head_dim;
  if (*rows == 0) return KAT_OK;   // and batch, tokens or heads may be anything
  if (q->rot_dim != 0) {
    if (q->cos_table == nullptr || q->sin_table == nullptr) return KAT_ERR_NULL_POINTER;
    if (q->positions == nullptr && q->table_rows < q->tokens) return KAT_ERR_BAD_SHAPE;
  }
  *vec = q->head_dim % 16 == 0 && q->head_dim <= kVecMaxHeadDim && q->rot_dim % 16 == 0 &&
         aligned16(q->cos_table) && aligned16(q->sin_table);
  const int per16 = 16 / elem_size(q->dtype);
  for (int i = 0; i < count; ++i) {
    const kat_head_stream& s = streams[i];
    Stream& d = p->s[i];
    if (d.rows != 0) {
      if (s.out == nullptr || (backward ? s.dy == nullptr : s.x == nullptr))
        return KAT_ERR_NULL_POINTER;
      for (int k = 0; k < 3; ++k) {
        if (s.out_stride[k] % per16 != 0 || (s.x != nullptr && s.x_stride[k] % per16 != 0) ||
            (backward && s.dy_stride[k] % per16 != 0))
          *vec = false;
      }
      if (!aligned16(s.x) || !aligned16(s.out) || (backward && !aligned16(s.dy))) *vec = false;
    }
    d.x = s.x;
    d.dy = s.dy;
    d.out = s.out;
    d.weight = s.weight;
    for (int k = 0; k < 3; ++k) {
      d.xs[k] = s.x_stride[k];
      d.ds[k] = s.dy_stride[k];
      d.os[k] = s.out_stride[k];
    }
    d.heads = divider(s.heads > 0 ? uint32_t(s.heads) : 1u);
  }
  p->tokens = divider(uint32_t(q->tokens));
  p->rot_dim = q->rot_dim;
  p->weight_dtype = q->weight_dtype;
  p->eps = q->eps;
  p->inv_dim = 1.0f / float(q->head_dim);
  p->cos_table = q->cos_table;
  p->sin_table = q->sin_table;
  p->table_rows = q->table_rows;
  p->positions = q->positions;
  p->ps[0] = q->position_stride[0];
  p->ps[1] = q->position_stride[1];
  return KAT_OK;
}

int lanes_of(int head_dim) { return head_dim <= 32 ? 2 : head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16; }

template <typename K>
int launch_ring(K kernel, uint32_t smem, const Params& p, dim3 grid, cudaStream_t st) {
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) !=
          cudaSuccess)
    return KAT_ERR_CUDA;
  kernel<<<grid, kThreads, smem, st>>>(p);
  return KAT_OK;
}
template <typename T, int LANES, bool INTER>
int launch_vec(const Params& p, bool backward, dim3 grid, cudaStream_t st) {
  return backward ? launch_ring(kat_head_bwd_kernel<T, LANES, INTER>, Ring<T, 4>::kBytes, p, grid, st)
                  : launch_ring(kat_head_fwd_kernel<T, LANES, INTER>, Ring<T, 2>::kBytes, p, grid, st);
}
template <typename T, bool INTER>
int launch_t(const Params& p, bool vec, bool backward, dim3 grid, cudaStream_t st) {
  if (!vec) {
    if (backward)
      kat_head_bwd_any_kernel<T, INTER>
          <<<grid, kThreads, size_t(kWarps) * p.head_dim * sizeof(float), st>>>(p);
    else
      kat_head_fwd_any_kernel<T, INTER><<<grid, kThreads, 0, st>>>(p);
    return KAT_OK;
  }
  switch (lanes_of(p.head_dim)) {
    case 2: return launch_vec<T, 2, INTER>(p, backward, grid, st);
    case 4: return launch_vec<T, 4, INTER>(p, backward, grid, st);
    case 8: return launch_vec<T, 8, INTER>(p, backward, grid, st);
    default: return launch_vec<T, 16, INTER>(p, backward, grid, st);
  }
}
template <typename T>
int launch_i(const Params& p, bool inter, bool vec, bool backward, dim3 grid, cudaStream_t st) {
  return inter ? launch_t<T, true>(p, vec, backward, grid, st)
               : launch_t<T, false>(p, vec, backward, grid, st);
}
int launch(const Params& p, int dtype, bool inter, bool vec, bool backward, dim3 grid,
           cudaStream_t st) {
  int rc = KAT_OK;
  switch (dtype) {
    case KAT_DTYPE_F32: rc = launch_i<float>(p, inter, vec, backward, grid, st); break;
    case KAT_DTYPE_F16: rc = launch_i<__half>(p, inter, vec, backward, grid, st); break;
    default: rc = launch_i<__nv_bfloat16>(p, inter, vec, backward, grid, st); break;
  }
  return cudaGetLastError() == cudaSuccess ? rc : KAT_ERR_CUDA;
}

int current_sms(int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KAT_ERR_CUDA;
  *sms = sm_count(dev);
  return *sms > 0 ? KAT_OK : KAT_ERR_CUDA;
}

// Blocks that hold every head of the longest stream at once, but no more than `most`; and each
// stream's run: as long as it leaves every group a turn.
uint32_t blocks_for(Params* p, int count, uint32_t rows, bool vec, uint32_t most) {
  const uint32_t per = vec ? kThreads / lanes_of(p->head_dim) : kWarps;
  const uint32_t want = (rows + per - 1) / per;
  const uint32_t blocks = want < most ? want : most;
  for (int i = 0; i < count; ++i) {
    p->s[i].run = kMaxRun;
    while (p->s[i].run > 1 && p->s[i].rows / p->s[i].run < blocks * per) p->s[i].run /= 2;
  }
  return blocks;
}

}  // namespace

extern "C" {

int kat_qk_norm_rope_fwd(const kat_head_problem* problem, const kat_head_stream* streams,
                         int32_t count, void* stream) {
  Params p{};
  bool vec = false;
  uint32_t rows = 0;
  if (int st = make_params(problem, streams, count, false, &p, &vec, &rows)) return st;
  if (rows == 0) return KAT_OK;
  int sms = 0;
  if (int st = current_sms(&sms)) return st;
  const dim3 grid(blocks_for(&p, count, rows, vec, uint32_t(sms) * kFwdBlocksPerSm),
                  uint32_t(count));
  return launch(p, problem->dtype, problem->interleaved != 0, vec, false, grid,
                static_cast<cudaStream_t>(stream));
}

size_t kat_qk_norm_rope_bwd_workspace_bytes(int32_t head_dim, int32_t count, int device) {
  if (head_dim < 1 || head_dim > kMaxHeadDim || count < 1 || count > KAT_MAX_HEAD_STREAMS)
    return 0;
  const int sms = sm_count(device);
  return sms <= 0 ? 0 : size_t(count) * sms * kBwdBlocksPerSm * head_dim * sizeof(float);
}

int kat_qk_norm_rope_bwd(const kat_head_problem* problem, const kat_head_stream* streams,
                         int32_t count, void* workspace, size_t workspace_bytes, void* stream) {
  Params p{};
  bool vec = false;
  uint32_t rows = 0;
  if (int st = make_params(problem, streams, count, true, &p, &vec, &rows)) return st;
  bool sums = false;
  for (int i = 0; i < count; ++i) sums |= p.s[i].dweight != nullptr && p.s[i].rows != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int sms = 0;
  if (rows != 0)
    if (int rc = current_sms(&sms)) return rc;
  const dim3 grid(blocks_for(&p, count, rows, vec, uint32_t(sms) * kBwdBlocksPerSm),
                  uint32_t(count));
  if (sums && (workspace == nullptr || !aligned16(workspace) ||
               workspace_bytes < size_t(count) * grid.x * p.head_dim * sizeof(float)))
    return KAT_ERR_WORKSPACE;
  for (int i = 0; i < count; ++i) {
    if (p.s[i].dweight == nullptr || p.s[i].rows != 0) continue;
    // a sum over no heads
    if (cudaMemsetAsync(p.s[i].dweight, 0, size_t(p.head_dim) * sizeof(float), st) != cudaSuccess)
      return KAT_ERR_CUDA;
    p.s[i].dweight = nullptr;
  }
  if (rows == 0) return KAT_OK;
  p.partial = static_cast<float*>(workspace);
  if (int rc = launch(p, problem->dtype, problem->interleaved != 0, vec, true, grid, st))
    return rc;
  if (sums) {
    kat_head_dweight_kernel<<<dim3((p.head_dim + 31) / 32, uint32_t(count)), 1024, 0, st>>>(
        p, int(grid.x));
    if (cudaGetLastError() != cudaSuccess) return KAT_ERR_CUDA;
  }
  return KAT_OK;
}

}  // extern "C"
