/* lattice_logits.h -- C-ABI of the operators over a model's logits (liblt.so).
 *
 * Beside the decoders, which find the best paths of a lattice under a linear
 * model (lattice_decode.h), these take the logits a neural model gives over a
 * vocabulary or a tag set:
 *   lt_top_logits        a row's k best logits and its log-sum-exp
 *   lt_distill_forward   the loss of a student's logits against a teacher's
 *   lt_distill_backward  top logits, its gradient,
 *   lt_distill_fused     and both in one pass
 *   lt_verify_draft      which drafted tokens a target's probabilities accept,
 *                        from given random numbers, and the token that follows
 *
 * Conventions: every pointer but `stream` (a hipStream_t, NULL for the null
 * stream) is device memory of the device the rows name; the calls queue
 * kernels on the stream and return -- they neither allocate, copy nor
 * synchronise, and may be captured into a graph.  Scratch memory is the
 * caller's: a buffer of at least lt_*_workspace bytes, 16 B aligned, that no
 * other call uses until this one's kernels are complete (its contents need
 * not be kept nor cleared; NULL where 0 bytes are needed).  The stream must be of the same device and of the
 * HIP runtime this library is bound to (lt_hip_library).  Calls may be made
 * from several threads at once.  Errors as in lattice_decode.h (lt_status,
 * lt_last_error).
 */
#ifndef LATTICE_LOGITS_H
#define LATTICE_LOGITS_H

#include <stdint.h>
#include "lattice_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define LT_F32 0
#define LT_F16 1
#define LT_BF16 2

#define LT_MAX_VOCAB (1 << 30)
#define LT_MAX_TOP 256     /* largest k of lt_top_logits, entries of a teacher's row */

/* Rows of logits: row r starts at element (r / inner) * stride_outer +
 * (r % inner) * stride_inner of data; its vocab elements are adjacent.  (So
 * logits[:, :-1] of a [batch, time, vocab] tensor need no copy.)  Nothing
 * outside the rows is read. */
typedef struct {
  const void* data;
  int32_t dtype;          /* LT_F32, LT_F16, LT_BF16 */
  int32_t device;         /* HIP device ordinal of every pointer of the call */
  int64_t rows;           /* >= 0; 0: the call does nothing */
  int64_t inner;          /* >= 1 */
  int64_t stride_outer;   /* in elements */
  int64_t stride_inner;
  int64_t vocab;          /* 1 .. LT_MAX_VOCAB */
} lt_rows;

/* Path of the HIP runtime library this library is bound to. */
const char* lt_hip_library(void);

/* ---- the k best logits of a row --------------------------------------------
 * ids[r*k + j], j = 0..k-1: the k largest logits of row r, largest first, ties
 * to the lowest index; a NaN counts as -inf in this order, -0 as 0.  values:
 * those logits, in the rows' type.  lse[r] = log sum_v exp(x_v / temperature): -inf
 * for a row of -inf, NaN if the row holds a NaN (and no +inf).
 * 1 <= k <= min(vocab, LT_MAX_TOP). */
int64_t lt_top_logits_workspace(const lt_rows* x, int32_t k);
lt_status lt_top_logits(const lt_rows* x, int32_t k, double temperature, void* values, int64_t* ids, float* lse,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* ---- distillation from a teacher's top logits ------------------------------
 * Row r of the student's logits z against K entries (ids[r*K + j],
 * top[r*K + j]) of the teacher's.  An id outside [0, vocab) is no entry.
 *   q_v = softmax(z / temperature)
 *   without top_lse: p_j = softmax of top / temperature over the entries
 *   with top_lse (the teacher's log-sum-exp at this temperature):
 *     p_j = exp(top_j / temperature - top_lse),  p_rest = max(0, 1 - sum p_j),
 *     q_rest = the q_v of every v that is no entry, summed
 *   loss = sum_j p_j (log p_j - log q_{id_j}) + p_rest (log p_rest - log q_rest)
 *     (the last term is left out, p_rest = 0, where the others are masked: each is
 *     -inf, or each the type's lowest value and more than 745 temperatures below the
 *     row's largest logit; else q_rest may be as small as logits can make it)
 *   d loss / d z_v = 1/temperature * (P q_v - sum_{id_j = v} p_j)       v an entry
 *                    1/temperature * (P - p_rest / q_rest) q_v         else
 *     with P = sum p_j + p_rest
 * A row without entries has loss 0 and gradient 0, whatever its logits, top and
 * top_lse hold.  One with entries whose logits hold a NaN or +inf, or are -inf
 * throughout, has loss NaN and gradient NaN, all of it.  An id that a row repeats counts once for each time.  The teacher is a constant.
 * 1 <= K <= LT_MAX_TOP. */
typedef struct {
  const void* ids;        /* [rows][entries] int32 or int64 */
  const void* top;        /* [rows][entries] */
  const float* top_lse;   /* [rows] or NULL */
  int32_t entries;
  int32_t ids_bytes;      /* 4 or 8 */
  int32_t top_dtype;      /* LT_F32, LT_F16, LT_BF16 */
} lt_teacher;

#define LT_DISTILL_STATS 4   /* floats a row that the forward leaves for the backward */

/* loss[rows]; stats[rows * LT_DISTILL_STATS], 16 B aligned. */
int64_t lt_distill_workspace(const lt_rows* z, int32_t entries);
lt_status lt_distill_forward(const lt_rows* z, const lt_teacher* t, double temperature, float* loss, float* stats,
                             void* workspace, int64_t workspace_bytes, void* stream);
/* grad: rows as z (its data, strides; same dtype and vocab) =
 * scale * weight[r * weight_stride] * d loss_r / d z; weight NULL: 1.
 * stats as the forward of the same arguments left them.  weight_stride 0 or 1.
 * No row of grad overlaps a row of z or another of its own. */
lt_status lt_distill_backward(const lt_rows* z, const lt_teacher* t, double temperature, const float* stats,
                              double scale, const float* weight, int64_t weight_stride, const lt_rows* grad,
                              void* stream);
/* Both at once. */
lt_status lt_distill_fused(const lt_rows* z, const lt_teacher* t, double temperature, double scale,
                           const float* weight, int64_t weight_stride, float* loss, const lt_rows* grad,
                           void* workspace, int64_t workspace_bytes, void* stream);

/* ---- verification of drafted tokens ----------------------------------------
 * target: rows = batch * (drafts + 1), row b * (drafts + 1) + i the target's
 * logits at the place of drafted token i of sequence b.  draft: rows = batch *
 * drafts, the logits that token i was drawn from, or NULL where the drafter
 * was certain of its tokens (q = 1 at the token).  With p, q = softmax of
 * those rows / temperature and n = lengths[b] (or drafts):
 *   a = the first i < n with accept_u[b, i] * q_i(x_i) >= p_i(x_i), else n
 *       (an id outside [0, vocab) has p = 0: it is never accepted)
 *   w = p_n if a = n, else max(p_a - q_a, 0), or p_a where that is 0 throughout
 *   token = the lowest v with w_v > 0 and w_0 + ... + w_v > sample_u[b] * sum w,
 *           else the last with w_v > 0; -1 if p_a is empty (a row of -inf)
 *   tokens[b] = x_0 .. x_{a-1}, token, -1 ...  [drafts + 1];  accepted[b] = a
 * Logits are finite or -inf (a NaN counts as -inf); a probability below 2^-1000 of
 * its row's largest counts as 0.  Rows past lengths[b] are not read; lengths are
 * taken as within [0, drafts].
 * Sums that decide the token are held in 64 bits. */
typedef struct {
  const lt_rows* target;
  const lt_rows* draft;       /* or NULL; dtype and vocab as target's */
  const void* ids;            /* [batch][drafts] int32 or int64 */
  const float* accept_u;      /* [batch][drafts], in [0, 1) */
  const float* sample_u;      /* [batch], in [0, 1) */
  const int32_t* lengths;     /* [batch] or NULL */
  int64_t batch;
  int32_t drafts;             /* >= 0 */
  int32_t ids_bytes;          /* 4 or 8 */
} lt_draft;
#define LT_MAX_DRAFTS 256

int64_t lt_verify_workspace(const lt_draft* d);
lt_status lt_verify_draft(const lt_draft* d, double temperature, int64_t* tokens, int64_t* accepted, void* workspace,
                          int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LATTICE_LOGITS_H */
