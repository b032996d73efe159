/*
 * hstu_recurrent.h -- C ABI of libhstu_recurrent.so: a gated linear recurrence over jagged sequences, which takes the attention's
 * place between the producer of u, v, q, k and the consumer, its step for single rows, and what stands between two layers (norm of
 * the block's output, gate, dropout, scale, residual, norm for the next block), for gfx950 (MI355X).
 *
 * Plain pointers and sizes; device pointers on the current HIP device; asynchronous on the stream given.  Nothing is
 * allocated and nothing read back to the host.  Index arrays hold int32 or int64 as the flag beside each says.  Row strides are in
 * elements, any that are not negative (in the recurrence up to 2^24); the columns of a row lie side by side.  Pointers are aligned to their elements (tensors are read in
 * wider pieces where their addresses and strides allow it).
 *
 * Status codes: 0 ok; negative values as in hstu_hip.h (-1 NULL pointer, -2 dtype, -4 alignment, -5 shape, -6 unsupported,
 * -7 launch failure, see hstu_recurrent_last_error(), -8 not a gfx950 device).
 */
#ifndef HSTU_RECURRENT_H_
#define HSTU_RECURRENT_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version, major*10000 + minor*100 + patch, and the text of the last HIP error seen by this thread ("" if none). */
int hstu_recurrent_version(void);
const char* hstu_recurrent_last_error(void);

/*
 * ---- The recurrence ----
 *
 * For every column c and every row t of a sequence, in fp32:
 *     z = rate * log(1 + exp(decay_c)) * sigmoid(decay_gate_t),  a = exp(-z)
 *     h_t = a * h_{t-1} + sqrt(1 - a^2) * sigmoid(input_gate_t) * x_t
 * h in front of a sequence's first row is initial_state[b], or 0.  out_t is h_t rounded to its type, final_state[b] the last h of the
 * sequence (its initial state where it has no rows), not rounded.  Where decay_gate is so low that its sigmoid is 0, a row of finite x leaves the state as it is.
 * A column with an infinity or a NaN is not finite from that row to the end of its sequence; other columns and sequences are not touched by it.
 * Rows behind the last sequence become zero.  seq_offsets begin at 0 and do not decrease; nothing is read or written out of
 * bounds where they do, but the results are no one's.
 */
typedef struct HstuRecurrenceArgs {
    const void* x;              /* [rows, width] */
    const void* decay_gate;     /* [rows, width] */
    const void* input_gate;     /* [rows, width] */
    int64_t x_row_stride, decay_gate_row_stride, input_gate_row_stride;
    void* out;                  /* [rows, width] dense, none of the inputs' memory; unused by the backward */
    const void* decay;          /* [width], fp32 or the type of x */
    int32_t decay_f32;
    float rate;                 /* finite, > 0 */
    const void* seq_offsets;    /* [batch + 1] */
    int32_t seq_offsets_i64;
    int32_t batch;              /* at least 1 */
    int64_t rows;
    int32_t width;
    int32_t dtype;              /* HstuDtype: bf16, fp16 or fp32 */
    const float* initial_state; /* [batch, width] dense, or NULL */
    float* final_state;         /* [batch, width] dense, or NULL: not wanted; unused by the backward */
    float* saved;               /* hstu_recurrent_scan_saved_bytes() bytes that the backward reads, or NULL: there is none to come */
    void* workspace;            /* hstu_recurrent_scan_workspace_bytes() bytes, 16-byte aligned; of the forward alone */
    int64_t workspace_bytes;
} HstuRecurrenceArgs;

/* What calls with these arguments need.  The forward's workspace goes by whether `saved` is NULL, so that is set first. */
size_t hstu_recurrent_scan_workspace_bytes(const HstuRecurrenceArgs* args);
size_t hstu_recurrent_scan_saved_bytes(const HstuRecurrenceArgs* args);
int hstu_recurrent_scan(const HstuRecurrenceArgs* args, void* stream);

/* Gradients from those of out and final_state (either may be NULL: zero).  `args` as in the forward call, `saved` included.  Each result may be
 * NULL: not wanted.  The decays' gradient is summed over a tile's rows in fp32 and over tiles in 64 bits, in an order that depends on
 * the sizes alone. */
typedef struct HstuRecurrenceGrads {
    const void* d_out;          /* [rows, width] */
    int64_t d_out_row_stride;
    const float* d_final_state; /* [batch, width] dense */
    void* d_x;                  /* [rows, width] dense, as the next two */
    void* d_decay_gate;
    void* d_input_gate;
    void* d_decay;              /* [width], in the type of decay */
    float* d_initial_state;     /* [batch, width] dense */
    void* workspace;            /* hstu_recurrent_scan_bwd_workspace_bytes() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} HstuRecurrenceGrads;

size_t hstu_recurrent_scan_bwd_workspace_bytes(const HstuRecurrenceArgs* args);
int hstu_recurrent_scan_bwd(const HstuRecurrenceArgs* args, const HstuRecurrenceGrads* grads, void* stream);

/*
 * One row for each of `rows` sequences: row r goes on from state slots[r] (-1: from nothing, zeros), and its new state is put into
 * new_slots[r] (-1: into none).  Without slots row r has state r; without new_slots they are slots.  A row whose slot is neither -1 nor one of the
 * states comes out NaN and is not put anywhere; nor is one whose new slot is not one.  No state may be put twice in a call, and none that
 * another row of the call reads; the states' memory is none of the other arguments'.
 */
typedef struct HstuRecurrenceStepArgs {
    const void* x;              /* [rows, width] */
    const void* decay_gate;
    const void* input_gate;
    int64_t x_row_stride, decay_gate_row_stride, input_gate_row_stride;
    void* out;                  /* [rows, width] dense */
    const void* decay;          /* [width], fp32 or the type of x */
    int32_t decay_f32;
    float rate;
    float* states;              /* [state_rows, width], changed in place */
    int64_t state_rows, state_row_stride;
    const void* slots;          /* [rows] or NULL */
    const void* new_slots;      /* [rows] or NULL */
    int32_t slots_i64, new_slots_i64;
    int64_t rows;
    int32_t width;
    int32_t dtype;
} HstuRecurrenceStepArgs;

int hstu_recurrent_step(const HstuRecurrenceStepArgs* args, void* stream);

/*
 * ---- Between two blocks ----
 *
 * For every row, in fp32:
 *     n = norm(y) * post_weight + post_bias           (n = y where post_weight is NULL)
 *     d = dropout(act(gate) * n)                      (act(gate) = 1 where gate is NULL)
 *     s = x + scale * d                               (scale = 1 where it is NULL)
 *     out = s,  normed = norm(s) * pre_weight + pre_bias    (s not rounded; pre_weight NULL: no normed)
 * norm(v) = v / sqrt(mean(v^2) + eps), or with layer_norm (v - mean v) / sqrt(var v + eps).  act: 0 gate itself, 1 its sigmoid, 2 gate * sigmoid(gate).
 * Dropout keeps element row * width + column where word element % 4 of Philox4x32-10 (counter (element / 4, offset), key seed)
 * is at least floor(p * 2^32), and divides it by 1 - p.  Nothing of it is stored: the backward computes the words again.
 */
typedef struct HstuResidualNormArgs {
    const void* x;              /* [rows, width] */
    const void* y;
    const void* gate;           /* or NULL */
    int64_t x_row_stride, y_row_stride, gate_row_stride;
    const void* post_weight;    /* [width] of the same type, or NULL, as the next four */
    const void* post_bias;
    const void* scale;
    const void* pre_weight;
    const void* pre_bias;
    void* out;                  /* [rows, width] dense; unused by the backward, as normed */
    void* normed;
    float eps;                  /* finite, not negative; below 2^-126 as 0: a row whose v^2 has a mean of 0 in fp32 is NaN */
    int32_t layer_norm;
    int32_t gate_activation;
    int32_t dtype;              /* HstuDtype: bf16, fp16 or fp32 */
    int64_t rows;
    int32_t width;              /* at most 8192 */
    double dropout_ratio;       /* 0: none; less than 1 */
    uint64_t dropout_seed, dropout_offset;
} HstuResidualNormArgs;

int hstu_recurrent_residual_norm(const HstuResidualNormArgs* args, void* stream);

/* Gradients from those of out and normed (either may be NULL: zero); statistics and dropout are computed again.  Each result may be NULL: not wanted.
 * Parameters' gradients are summed over rows by each lane in fp32 and over the lanes in 64 bits, in an order that depends on the sizes alone. */
typedef struct HstuResidualNormGrads {
    const void* d_out;          /* [rows, width] */
    const void* d_normed;       /* [rows, width]; not read where pre_weight is NULL */
    int64_t d_out_row_stride, d_normed_row_stride;
    void* d_x;                  /* [rows, width] dense, as the next two */
    void* d_y;
    void* d_gate;
    void* d_post_weight;        /* [width] */
    void* d_post_bias;
    void* d_scale;
    void* d_pre_weight;
    void* d_pre_bias;
    void* workspace;            /* hstu_recurrent_residual_norm_bwd_workspace_bytes() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} HstuResidualNormGrads;

size_t hstu_recurrent_residual_norm_bwd_workspace_bytes(const HstuResidualNormArgs* args);
int hstu_recurrent_residual_norm_bwd(const HstuResidualNormArgs* args, const HstuResidualNormGrads* grads, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* HSTU_RECURRENT_H_ */
