/*
 * esgd_ops.h — operators of a language model's training step around its matrix products:
 * embedding lookup, the order of tokens by expert, and the distillation loss, each with its
 * gradient.  They make the gradients that the schedules of esgd.h reduce.  No counterpart in
 * the reference, whose models are TF graphs.
 *
 * Conventions of esgd.h: plain device pointers and sizes, an int status, the message in
 * esgd_last_error(), stream NULL = the library's stream of the current device,
 * ESGD_STREAM_NULL = the legacy default stream.  Every call queues its kernels on that stream
 * and returns; none allocates, synchronises or keeps anything, so all of them can be captured
 * into a graph.  Calls that need scratch memory take it from the caller (`work`, whose size the
 * matching *_work function gives); it is free again once the stream has passed the call, and two
 * calls that may run at once need two of them.
 *
 * Floating types: ESGD_FLOAT, ESGD_BF16, ESGD_HALF.  Sums, softmax statistics and products are
 * fp32 whatever the types, rounded once at the store.  Results do not depend on the order in
 * which workgroups run: the same call gives the same bits.  A row is `width` elements next to
 * each other; where a pitch (elements from row to row) is taken, rows may stand further apart, at
 * any alignment that the element's own type allows.
 */
#ifndef ESGD_OPS_H
#define ESGD_OPS_H

#include "esgd.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ESGD_HALF 17 /* IEEE binary16: the operators of this header only */

/* ---- embedding ----
 * out[t] = scale * table[token[t]], `n` rows.  token: int32 or int64 (token_bits 32 / 64), next
 * to each other.  A token outside [0, rows) -- padding, say -1 -- reads as a row of zeros.
 * table_type FLOAT with any out_type, or both the same. */
int esgd_embedding(int table_type, const void *table, int64_t table_pitch, int64_t rows, int64_t width,
                   int token_bits, const void *token, int64_t n, float scale, int out_type, void *out,
                   int64_t out_pitch, void *stream);

/* grad_table[v] (rows x width, contiguous) = scale * sum of grad[t] over the t with token[t] == v;
 * tokens outside [0, rows) and those equal to skip_token give nothing (skip_token < 0: none).
 * accumulate 0: every row is written, zeros where no token names it; 1: the sums are added to
 * grad_table's rows and rows that no token names are neither read nor written.  Same sums in
 * the same order at every call: no atomics on floats.  n < 2^31 - 65536, rows < 2^31 - 1, width < 2^28,
 * n * (width up to the next multiple of 256) < 2^35. */
int esgd_embedding_grad_work(int64_t n, int64_t rows, int64_t width, size_t *bytes);
int esgd_embedding_grad(int grad_type, const void *grad, int64_t grad_pitch, int64_t n, int64_t width,
                        int token_bits, const void *token, int64_t skip_token, float scale, int table_type,
                        void *grad_table, int64_t rows, int accumulate, void *work, size_t work_bytes,
                        void *stream);

/* ---- tokens by expert ----
 * expert: tokens x choices, int32 or int64.  The pairs (t, j) sorted by expert, equal experts in
 * the order of (t, j): offsets[e] .. offsets[e + 1] are expert e's places (`experts` + 1 int32),
 * slots[t * choices + j] (int32) is the pair's place.  A pair whose expert is outside
 * [0, experts) is dropped: its place p lies behind every expert's and its slot is -1 - p. */
int esgd_expert_sort_work(int64_t pairs, int64_t experts, size_t *bytes);
int esgd_expert_sort(int expert_bits, const void *expert, int64_t tokens, int64_t choices, int64_t experts,
                     int32_t *offsets, int32_t *slots, void *work, size_t work_bytes, void *stream);

/* rows[slot(t, j)] = x[t]; the places of dropped pairs are filled with zeros.  rows:
 * (tokens * choices) x width, contiguous, wholly written. */
int esgd_expert_dispatch(int type, const void *x, int64_t x_pitch, int64_t tokens, int64_t choices,
                         int64_t width, const int32_t *slots, void *rows, void *stream);
/* grad_x[t] = sum over j of grad_rows[slot(t, j)], in the order of j; dropped pairs give nothing */
int esgd_expert_dispatch_grad(int type, const void *grad_rows, int64_t grad_pitch, int64_t tokens,
                              int64_t choices, int64_t width, const int32_t *slots, void *grad_x,
                              void *stream);
/* out[t] = sum over j of weights[t, j] * rows[slot(t, j)], in the order of j.  weights: fp32,
 * contiguous.  The weights of dropped pairs and the rows at their places change nothing, whatever
 * they are, but have to be memory that can be read. */
int esgd_expert_combine(int type, const void *rows, int64_t rows_pitch, int64_t tokens, int64_t choices,
                        int64_t width, const int32_t *slots, const float *weights, void *out, void *stream);
/* grad_rows[slot(t, j)] = weights[t, j] * grad[t] (zeros for dropped pairs; wholly written) and
 * grad_weights[t, j] = <grad[t], rows[slot(t, j)]> (0 for dropped pairs; what stands
 * in their weights and rows changes nothing, but has to be memory that can be read) */
int esgd_expert_combine_grad(int type, const void *grad, int64_t grad_pitch, const void *rows,
                             int64_t rows_pitch, int64_t tokens, int64_t choices, int64_t width,
                             const int32_t *slots, const float *weights, void *grad_rows,
                             float *grad_weights, void *stream);

/* ---- distillation from a teacher's top logits ----
 * Per row: p = softmax(top_logits / temperature) over the entries whose top_index is in
 * [0, vocab), q = softmax(logits / temperature) over the whole row,
 *   loss = temperature^2 * sum_k p_k (log p_k - log q[top_index_k]).
 * An index that stands there twice counts twice.  A row without any entry of finite or +infinite
 * teacher logit has loss 0 and gradient 0, whatever its logits are (they have to be memory that can
 * be read).
 * stats (4 floats a row): what the gradient needs of the pass. */
#define ESGD_DISTILL_TOP_MAX 1024
int esgd_distill_work(int64_t n, int64_t vocab, size_t *bytes);
int esgd_distill_loss(int type, const void *logits, int64_t pitch, int64_t n, int64_t vocab, int top_type,
                      const void *top_logits, int index_bits, const void *top_index, int64_t top,
                      float temperature, float *loss, float *stats, void *work, size_t work_bytes,
                      void *stream);
/* grad_logits (n x vocab, contiguous) = row_grad[r * row_grad_pitch] * d loss[r] / d logits */
int esgd_distill_grad(int type, const void *logits, int64_t pitch, int64_t n, int64_t vocab, int top_type,
                      const void *top_logits, int index_bits, const void *top_index, int64_t top,
                      float temperature, const float *stats, const float *row_grad, int64_t row_grad_pitch,
                      void *grad_logits, void *stream);
/* both at once where row_grad is known beforehand */
int esgd_distill_loss_grad(int type, const void *logits, int64_t pitch, int64_t n, int64_t vocab,
                           int top_type, const void *top_logits, int index_bits, const void *top_index,
                           int64_t top, float temperature, const float *row_grad, int64_t row_grad_pitch,
                           float *loss, float *stats, void *grad_logits, void *work, size_t work_bytes,
                           void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ESGD_OPS_H */
