/*
 * hstu_cache.h -- C ABI of libhstu_cache.so: rotated positions with norms per head, a paged K/V cache held in 4 bits and
 * the attention that reads it, for gfx950 (MI355X).
 *
 * The steps, in the order a layer takes them: `hstu_cache_norm_rope` between the producer of q, k, v and the attention
 * (forward and backward); `hstu_cache_append` puts new K and V rows into the pages of a cache, normed and rotated on the
 * way; `hstu_cache_attention` is the cached form of the HSTU attention (hstu_hip.h, delta_size > 0) on that cache;
 * `hstu_cache_read` gives rows of it back as values for the operators that read 16-bit K and V.
 *
 * Plain pointers and sizes; device pointers on the current HIP device; asynchronous on the stream given.  Nothing is
 * allocated and nothing read back to the host.  Index arrays hold int32 or int64 as the flag beside each says.  Strides are
 * in elements, innermost stride 1; rows and heads of K, V, q and their gradients lie on 16-byte boundaries.
 *
 * Status codes: 0 ok; negative values as in hstu_hip.h (-1 NULL pointer, -2 dtype, -3 head dim, -4 alignment, -5 shape,
 * -6 unsupported, -7 launch failure, see hstu_cache_last_error(), -8 not a gfx950 device).
 */
#ifndef HSTU_CACHE_H_
#define HSTU_CACHE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version, major*10000 + minor*100 + patch, and the text of the last HIP error seen by this thread ("" if none). */
int hstu_cache_version(void);
const char* hstu_cache_last_error(void);

/*
 * ---- Norms of q and k for each head, and the position rotation, in one pass ----
 *
 * For every row r and head of x (q or k, the weight of its own):
 *     n = x / sqrt(mean(x^2) + eps) * weight          (n = x where the weight is NULL)
 *     y = n, its first `rotary` columns turned by the angles of position positions[r]:
 *         half-split   pairs (i, i + rotary / 2):  y_i = n_i cos_i - n_j sin_i,  y_j = n_j cos_i + n_i sin_i
 *         interleaved  pairs (2 i, 2 i + 1)
 * with cos_i = table[p][i] and sin_i = table[p][rotary / 2 + i].  Everything in fp32, rounded once.
 * A row whose position lies outside of the table becomes NaN.
 */
typedef struct HstuNormRopeArgs {
    const void* q;             /* [rows, q_heads, dim]; NULL: no q */
    const void* k;             /* [rows, k_heads, dim]; NULL: no k */
    int64_t q_row_stride, q_head_stride, k_row_stride, k_head_stride;
    void* q_out;               /* [rows, q_heads, dim] dense; unused by the backward */
    void* k_out;
    const void* q_weight;      /* [dim] of the same type, or NULL: no norm */
    const void* k_weight;
    float eps;
    const void* positions;     /* [rows]; needed where rotary > 0 */
    int32_t positions_i64;
    int32_t rotary;            /* 0: no rotation; half-split: a multiple of 16, interleaved: of 8; at most dim */
    int32_t interleaved;
    const float* table;        /* [table_rows, rotary] */
    int64_t table_rows;
    int64_t rows;
    int32_t q_heads, k_heads;
    int32_t dim;               /* a multiple of 8, at most 512 */
    int32_t dtype;             /* HstuDtype: bf16, fp16 or fp32 */
} HstuNormRopeArgs;

int hstu_cache_norm_rope(const HstuNormRopeArgs* args, void* stream);

/* Gradients from those of the outputs; statistics are recomputed from q and k.  A weight's gradient is summed over rows and
 * heads, by each lane in fp32 and over the lanes in 64 bits, in an order that depends on the sizes alone; its workspace is needed where
 * either is asked for. */
typedef struct HstuNormRopeGrads {
    const void* dq_out;        /* [rows, q_heads, dim]; NULL where q is */
    const void* dk_out;
    int64_t dq_out_row_stride, dq_out_head_stride, dk_out_row_stride, dk_out_head_stride;
    void* dq;                  /* [rows, q_heads, dim] dense */
    void* dk;
    void* dq_weight;           /* [dim] where q_weight is there, or NULL: not wanted */
    void* dk_weight;
    void* workspace;           /* hstu_cache_norm_rope_bwd_workspace_bytes() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} HstuNormRopeGrads;

size_t hstu_cache_norm_rope_bwd_workspace_bytes(const HstuNormRopeArgs* args);
int hstu_cache_norm_rope_bwd(const HstuNormRopeArgs* args, const HstuNormRopeGrads* grads, void* stream);

/*
 * ---- The cache ----
 *
 * Pages of `page_size` positions, the positions of one head side by side.  A row (one position, one head) is `dim` codes of
 * 4 bits, two to a byte, the even column in the low half, and a pair (step, lowest value) in the type of K and V; the value
 * of a column is  lowest + step * code.  Row x in that type becomes
 *     lowest = min x,  step = (max x - min x) / 15 rounded to the type,  code = (x - lowest) / step rounded to the nearest
 * (ties to even) and held within 0 .. 15; code 0 throughout where step is 0.  The difference and the quotient are rounded to fp32.  A row with a NaN or an infinity, or whose step
 * the type does not hold, becomes NaN: step and lowest value both.
 * Position i of sequence b lies in page page_table[b][i / page_size].
 */
typedef struct HstuPagedCache {
    void* k_codes;             /* [pages, heads, page_size, dqk / 2] bytes, dense, 16-byte aligned, as the next three */
    void* k_scales;            /* [pages, heads, page_size, 2] */
    void* v_codes;             /* [pages, heads, page_size, dv / 2] */
    void* v_scales;            /* [pages, heads, page_size, 2] */
    int64_t pages;
    int32_t heads;
    int32_t page_size;         /* a power of two, 16 .. 1024 */
    int32_t dqk, dv;           /* 32, 64, 128 or 256 */
    int32_t dtype;             /* HstuDtype: bf16 or fp16 */
    const void* page_table;    /* [batch, table_columns], row stride in elements */
    int64_t table_row_stride;
    int32_t table_columns;
    int32_t page_table_i64;
    int32_t batch;
} HstuPagedCache;

/*
 * New rows into their pages: row seq_offsets[b] + i of k and v is position start[b] + i of sequence b (without seq_offsets:
 * row b * (rows / batch) + i).  K rows go through the norm and the rotation of hstu_cache_norm_rope, are rounded to their
 * type and then to 4 bits.  The angle is that of positions[row], or of the row's place in its sequence where positions is NULL.
 * Rows behind the last sequence are left alone; so is a row whose place lies outside of the page table or whose page is not one
 * of the cache's.  No two rows of a call may have one place.
 */
typedef struct HstuAppendArgs {
    const void* k;             /* [rows, heads, dqk] */
    const void* v;             /* [rows, heads, dv] */
    int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    int64_t rows;
    const void* start;         /* [batch] */
    const void* seq_offsets;   /* [batch + 1] or NULL */
    int32_t start_i64, seq_offsets_i64;
    const void* k_weight;      /* [dqk] or NULL */
    float eps;
    int32_t rotary, interleaved;
    const float* table;
    int64_t table_rows;
    const void* positions;     /* [rows] or NULL */
    int32_t positions_i64;
} HstuAppendArgs;

int hstu_cache_append(const HstuPagedCache* cache, const HstuAppendArgs* args, void* stream);

/*
 * Rows of the cache as values, rounded to its type: row seq_offsets[b] + i of k and v (dense [rows, heads, dim]) is position
 * start[b] + i of sequence b.  Rows behind the last sequence become zero; a row whose place has no page becomes NaN.
 */
int hstu_cache_read(const HstuPagedCache* cache, int64_t rows, const void* start, int32_t start_i64, const void* seq_offsets,
                    int32_t seq_offsets_i64, void* k, void* v, void* stream);

/*
 * ---- Attention over the cache ----
 *
 * out[b * delta_size + i] = sum_s M(p, s) * silu(alpha * <q, k_s>) / max_seq_len * v_s  for the newest delta_size positions
 * p = seq_lengths[b] - delta_size + i of every sequence, with the masks of the cached form (hstu_hip.h).  Head h of q reads head
 * h / (q_heads / heads) of the cache.  K and V enter as lowest + step * code, unrounded; silu(.) times a V row's step is rounded to
 * bf16 for the second product (to two bf16 words, 16 bits, where the type is fp16 or no more than eight rows of q, delta_size times
 * q_heads / heads, share a head), sums are in fp32 and rounded once.  Codes enter the
 * products with an offset of up to 128: sums over a row of |q|, or over the positions of |silu(.)| times a V row's step, of 2^120 and
 * more may overflow.
 * A row at a position before the first is zero.  A sequence that is longer than its row of the page table gives NaN.  Where one of its
 * pages is not one of the cache's, every row that sees a position on that page is NaN, and other rows of the sequence may be; pages that end
 * in front of the first position that any row of the call sees (behind a window) are not looked at.
 * The positions of a row block are cut into runs that `workspace` joins (kv_splits: 0 = automatic, else at most that many); the
 * order of the sums depends on the sizes of the call and the lengths alone.
 */
typedef struct HstuPagedAttentionArgs {
    const void* q;             /* [batch * delta_size, q_heads, dqk] */
    int64_t q_row_stride, q_head_stride;
    void* out;                 /* [batch * delta_size, q_heads, dv] dense */
    const void* seq_lengths;   /* [batch], the newest delta_size positions included */
    const void* num_targets;   /* [batch] or NULL */
    int32_t seq_lengths_i64, num_targets_i64;
    int32_t q_heads;           /* a multiple of the cache's heads */
    int32_t delta_size;
    int32_t max_seq_len;
    float alpha;
    int32_t max_attn_len, contextual_seq_len;
    int32_t kv_splits;
    void* workspace;           /* hstu_cache_attention_workspace_bytes() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} HstuPagedAttentionArgs;

size_t hstu_cache_attention_workspace_bytes(const HstuPagedCache* cache, const HstuPagedAttentionArgs* args);
int hstu_cache_attention(const HstuPagedCache* cache, const HstuPagedAttentionArgs* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* HSTU_CACHE_H_ */
