/* flashcqt_seq.h -- C ABI of the sequence operators (libflashcqt_seq.so) for MI355X (gfx950): what a model over
 * CQT frames is trained and run with, beside the transform itself (flashcqt.h, libflashcqt.so).
 *
 *   fcqt_head_norm_rotary[_bwd]   RMS norm of every head of q and k and their rotation by positions, in one pass
 *   fcqt_decay_attention          linear attention with a decay for each head, over whole sequences; run forwards
 *                                 or backwards in time it also gives its own gradients
 *   fcqt_decay_attention_step     the same for one token of every running sequence, states in a pool
 *   fcqt_adamw, fcqt_adamw_drawn, fcqt_adamw_read
 *                                 one AdamW step over many tensors, moments in 32 or in 8 bits
 *
 * Conventions, as in flashcqt.h: every buffer is device memory of the caller's, nothing is allocated; all work is
 * enqueued on `stream`, which may be under hipGraph capture; argument errors are found before any HIP call and
 * returned as FCQT_E* codes; no result is accumulated with atomics, so results are the same from call to call.
 * Strides are in elements. The innermost dimension of every tensor is contiguous. */
#ifndef FLASHCQT_SEQ_H
#define FLASHCQT_SEQ_H

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#include "flashcqt.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FCQT_SEQ_ABI_VERSION 2

/* element types */
#define FCQT_F32 0
#define FCQT_BF16 1
#define FCQT_F16 2

#define FCQT_SEQ_MAX_DIM 256   /* largest head dimension */
#define FCQT_DECAY_MAX_DIM 128 /* largest of attention over whole sequences: its states stay in registers */
#define FCQT_ROTARY_AXES 4     /* most position axes */

int fcqt_seq_abi_version(void);

/* text of the last HIP error this library saw, on any thread */
const char* fcqt_seq_last_hip_error(void);

/* ---- head norm with rotary positions ---- */

/* A [batch][tokens][heads][dim] tensor read in place. */
typedef struct fcqt_heads {
    const void* data;
    int64_t batch_stride, token_stride, head_stride;
    int32_t heads;
} fcqt_heads;

typedef struct fcqt_rotary {
    const float* positions;   /* [batch or 1][tokens][axes] */
    int64_t positions_batch;  /* elements from one row's positions to the next; 0: all rows share them */
    const float* freq;        /* [pairs] angle of each pair for a position of one */
    int32_t axes;             /* 1..FCQT_ROTARY_AXES, or 0: no rotation */
    int32_t ends[FCQT_ROTARY_AXES]; /* one past the last pair that each axis turns, ascending; the last is `pairs` */
    int32_t interleaved;      /* pairs are (2j, 2j+1); else (j, j + pairs) */
} fcqt_rotary;

/* q_out, k_out: contiguous [batch][tokens][heads][dim] of the inputs' type. wq, wk: [dim] fp32 or NULL (ones).
 * norm = 0 leaves the norm (and the weights) out. dim is a multiple of 8, at most FCQT_SEQ_MAX_DIM; 2 * pairs <=
 * dim; pairs that are not interleaved are a multiple of 4. */
int fcqt_head_norm_rotary(const fcqt_heads* q, const fcqt_heads* k, const fcqt_rotary* rot, const float* wq,
                          const float* wk, void* q_out, void* k_out, int64_t batch, int64_t tokens, int32_t dim,
                          int32_t dtype, int32_t norm, float eps, hipStream_t stream);

/* Gradients: gq, gk are those of the outputs; dq, dk (contiguous) those of the inputs, dw [2][dim] those of wq and
 * wk. partial: workspace of fcqt_head_norm_rotary_partial(...) floats. dw and partial may be NULL together. */
int64_t fcqt_head_norm_rotary_partial(int64_t batch, int64_t tokens, int32_t heads, int32_t dim, int32_t dtype);
int fcqt_head_norm_rotary_bwd(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* gq, const fcqt_heads* gk,
                              const fcqt_rotary* rot, const float* wq, const float* wk, void* dq, void* dk, float* dw,
                              float* partial, int64_t batch, int64_t tokens, int32_t dim, int32_t dtype, int32_t norm,
                              float eps, hipStream_t stream);

/* ---- linear attention with a decay for each head ---- */

/* Whole sequences: S_t = exp(log_decay) S_{t-1} + k_t v_t', o_t = scale q_t S_t, from `state` (NULL: zero) to `last`,
 * both contiguous [batch][hk][dk][dv] fp32. Heads are shared as in the step below. lengths: valid tokens of each row
 * (NULL: all; taken into 0..tokens); what lies past them is not used, o is zero there and `last` is the state at the
 * length. o: contiguous [batch][tokens][hq][dv]. q, k and v are read 16 bytes at a time: their places and strides are
 * multiples of that, token strides under 2^31 bytes / 64. dk and dv are multiples of 8, at most
 * FCQT_DECAY_MAX_DIM; batch at most 65535, tokens below 2^31 - 64. fp32 operands and states go through bf16 planes: a value
 * over bf16's largest, 3.38e38, or an infinite one makes NaN. workspace: fcqt_decay_attention_workspace(...) bytes (0: NULL
 * will do), ragged where lengths are given, with backward 0; for the gradients with 1, or with 2 where dlog_decay is among them. */
int64_t fcqt_decay_attention_workspace(int64_t batch, int64_t tokens, int32_t hq, int32_t hk, int32_t dk, int32_t dv,
                                       int32_t dtype, int32_t ragged, int32_t backward);
int fcqt_decay_attention(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v, const float* log_decay,
                         const int32_t* lengths, const float* state, float* last, void* o, void* workspace,
                         int64_t workspace_bytes, int64_t batch, int64_t tokens, int32_t dk, int32_t dv, int32_t dtype,
                         float scale, hipStream_t stream);

/* Its gradients, from go (that of o) and glast (that of `last`, or NULL): dq, dk, dv contiguous and of the inputs'
 * type, a shared head's summed over its query heads; dlog_decay [hk] and dstate fp32, or NULL where not wanted. starts:
 * the workspace as fcqt_decay_attention left it for the same arguments, or NULL. */
int fcqt_decay_attention_bwd(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v, const float* log_decay,
                             const int32_t* lengths, const float* state, const void* starts, const fcqt_heads* go,
                             const float* glast, void* dq, void* dk_, void* dv_, float* dlog_decay, float* dstate, void* workspace,
                             int64_t workspace_bytes, int64_t batch, int64_t tokens, int32_t dk, int32_t dv,
                             int32_t dtype, float scale, hipStream_t stream);

/* One token of `batch` sequences: S <- exp(log_decay) S + k v', o = scale q S. q [batch][hq], k, v [batch][hk] heads
 * (token_stride unused), hq a multiple of hk; query head h reads key head h / (hq / hk). state: [pool][hk][dk][dv] fp32; row b uses
 * state slots[b], or b where slots is NULL. A row whose slot is outside 0..pool-1 has no sequence: its o is zero and
 * no state changes. Two rows must not name the same slot. o: contiguous [batch][hq][dv]. dk and dv are multiples of
 * 8, at most FCQT_SEQ_MAX_DIM. */
int fcqt_decay_attention_step(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v, const float* log_decay,
                              float* state, const int32_t* slots, void* o, int64_t batch, int64_t pool, int32_t dk,
                              int32_t dv, int32_t dtype, float scale, hipStream_t stream);

/* ---- AdamW ---- */

/* A tensor and its moments. With 32-bit moments m and v are fp32 [n] and the scales NULL; with 8-bit ones they are
 * codes [n] with a scale for every FCQT_ADAMW_BLOCK elements. */
typedef struct fcqt_adamw_tensor {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    int64_t n;
} fcqt_adamw_tensor;

#define FCQT_ADAMW_BLOCK 256

/* The step's factors: m = b1 m + c1 g, v = b2 v + c2 g g, p = keep p - rate m / (root sqrt(v) + eps). */
typedef struct fcqt_adamw_factors {
    float b1, c1, b2, c2, keep, rate, root, eps;
} fcqt_adamw_factors;

/* `tensors` is host memory, read before the call returns. dtype: of p and g. grad_scale: NULL, or a device scalar
 * that every gradient is multiplied by first. Tensors of no elements are passed over. With bits = 8 every moment gets
 * its nearest code, which is not for many steps: a moment that a step changes by less than half a code's step stays. */
int fcqt_adamw(const fcqt_adamw_tensor* tensors, int64_t count, int32_t dtype, int32_t bits,
               const fcqt_adamw_factors* factors, const float* grad_scale, hipStream_t stream);

/* With 8-bit moments, over many steps: each code is one of its value's two neighbours, drawn by a hash of seed, step,
 * the tensor's place in the list and the element, so that m and v are kept on average. `step` is another one at each call. */
int fcqt_adamw_drawn(const fcqt_adamw_tensor* tensors, int64_t count, int32_t dtype, const fcqt_adamw_factors* factors,
                     const float* grad_scale, uint64_t seed, int64_t step, hipStream_t stream);

/* The values that 8-bit moments stand for: p and g of each tensor name fp32 [n] buffers for m and v. */
int fcqt_adamw_read(const fcqt_adamw_tensor* tensors, int64_t count, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FLASHCQT_SEQ_H */
