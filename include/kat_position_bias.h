/*
 * kat_position_bias.h — C ABI of the learned relative position bias by buckets in
 * libkat_rational.so (sm_100a): out[h, i, j] = table[bucket(i, j), h], and the table's gradient
 * d_table[b, h] = sum of dout[h, i, j] over all (i, j) of bucket b.
 *
 * Two kinds of bucket:
 *
 *   distance   bucket(i, j) = bucket_of[j - i - offset], looked up in an int32 table over the
 *              distances -reach .. reach (farther ones take the ends).  Equal distances must
 *              share a bucket only with neighbours: each bucket is one run of distances, given
 *              by run_begin / run_end (inclusive; INT32_MIN / INT32_MAX where it has no end).
 *              With `causal`, out is -infinity where j - i > offset and those cells take no part
 *              in the gradient, whatever dout holds there.
 *   index      bucket(i, j) from an int32 matrix [lq, ld], ld = lk rounded up to 8; cells of
 *              bucket num_buckets (padding, or no bias) are 0 and have no gradient.
 *
 * `out` is [heads, lq, ld] contiguous, ld = lk rounded up to 8, the columns behind lk are set to
 * zero: rows start at multiples of 16 bytes, as attention kernels read a mask.  dout has any
 * strides.  The table is [num_buckets, heads] contiguous; out and dout have their own types.
 * Gradients are sums in a fixed order, fp32 within runs and fp64 above them.
 *
 * The index gradient goes by segments: the rows are cut into slabs of whole rows of at most
 * KAT_BIAS_SLAB_CELLS padded cells; within a slab the cells are sorted by bucket and cut into
 * segments of one bucket each and at most KAT_BIAS_SEGMENT cells.
 *   cells       uint16 place in the slab (row in the slab * lk + column), segment by segment;
 *               padded_cells the same with rows of ld (the kernel takes what dout's rows are)
 *   seg_begin   [segments + 1] first cell of each segment; slab_begin [slabs + 1] first segment
 *   seg_place   [segments] each segment's place in the order of buckets; bucket_begin
 *               [num_buckets + 1] first place of each bucket
 *
 * The same rules as in kat_rational.h: nothing is allocated, work is enqueued on `stream` of the
 * current device, argument errors are reported before anything is enqueued.
 */
#ifndef KAT_POSITION_BIAS_H_
#define KAT_POSITION_BIAS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KAT_BIAS_SLAB_CELLS 16384
#define KAT_BIAS_SEGMENT 32

int kat_distance_bias_fwd(const void* table, int32_t table_dtype, int32_t num_buckets,
                          int32_t heads, const int32_t* bucket_of, int32_t reach, int64_t lq,
                          int64_t lk, int64_t offset, int32_t causal, void* out,
                          int32_t out_dtype, void* stream);

size_t kat_distance_bias_bwd_workspace_bytes(int32_t heads, int64_t lq, int64_t lk);

/* d_table [num_buckets, heads] of type table_dtype from dout with strides (head, row, column). */
int kat_distance_bias_bwd(const void* dout, int32_t dout_dtype, const int64_t* dout_stride,
                          int32_t num_buckets, int32_t heads, const int32_t* run_begin,
                          const int32_t* run_end, int64_t lq, int64_t lk, int64_t offset,
                          int32_t causal, void* d_table, int32_t table_dtype, void* workspace,
                          size_t workspace_bytes, void* stream);

int kat_index_bias_fwd(const void* table, int32_t table_dtype, int32_t num_buckets, int32_t heads,
                       const int32_t* index, int64_t lq, int64_t lk, void* out, int32_t out_dtype,
                       void* stream);

size_t kat_index_bias_bwd_workspace_bytes(int32_t heads, int64_t segments);

int kat_index_bias_bwd(const void* dout, int32_t dout_dtype, const int64_t* dout_stride,
                       int32_t num_buckets, int32_t heads, int64_t lq, int64_t lk,
                       const uint16_t* cells, const uint16_t* padded_cells,
                       const int32_t* seg_begin, int64_t segments, const int32_t* slab_begin,
                       int64_t slabs, int32_t slab_rows,
                       const int32_t* seg_place, const int32_t* bucket_begin, void* d_table,
                       int32_t table_dtype, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KAT_POSITION_BIAS_H_ */
