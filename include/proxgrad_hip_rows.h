/*
 * proxgrad_hip_rows.h -- smooth losses whose scores come in ROWS (one softmax per row), on libproxgrad_hip.so.
 *
 * proxgrad_hip.h evaluates losses of one score per sample (pg_loss_value_and_gradient).  The entry points here evaluate
 * losses of a whole row of scores per sample, for classifiers, re-rankers and routers fitted with the same iterations:
 * value_and_gradient(f, u) -> (f(u), grad f(u)) with u the rows one after another.  Same conventions as proxgrad_hip.h
 * (opaque context, device pointers, pg_status, work enqueued on the context's stream).  Apart from those headers and
 * versioned by itself: a host written against the boundary header alone needs nothing of this one.
 *
 * Element types: scores and gradients are PG_F32, PG_F64, PG_BF16 or PG_F16.  Arithmetic, softmax statistics and sums are
 * Float32 for the three narrow types and Float64 for PG_F64; the total over the rows is Float64; each gradient entry is
 * rounded to the scores' type once.
 *
 * Rows are `ld` elements apart (ld >= the row's length), elements of a row are adjacent, no alignment is asked for beyond
 * the element's own.  What lies between the rows is neither read nor written.  grad may be the scores' own buffer (same
 * pointer, same ld); any other overlap is not allowed.
 *
 * An entry point that is given f_out (host) synchronises the context's stream and stores f there; with f_out = NULL it
 * is asynchronous.  `value` (device, may be NULL) receives f as a Float32 (Float64 for PG_F64 scores).
 * Inside a capture (pg_ctx_capture_begin) f_out is not meaningful; a stream that is being captured by anybody else is refused.
 */
#ifndef PROXGRAD_HIP_ROWS_H
#define PROXGRAD_HIP_ROWS_H

#include "proxgrad_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* bumped with every change of this header's signatures or structs */
#define PG_ROWS_ABI_VERSION 1
int32_t pg_rows_abi_version(void);

enum { PG_BF16 = 2, PG_F16 = 3 }; /* beside PG_F32, PG_F64: understood by this header's entry points only */

/* ------------------------------------------------------------------ distillation from a teacher's top logits ---- */
/* Scores x (rows x classes), teacher's listed logits t at classes i (rows x top; an entry with index -1 is absent),
 * temperature T, per-row weights w (NULL: ones; >= 0):  z = x / T, log q = z - log sum exp z, S = the listed classes,
 *   teacher_lse == NULL:  p_k = exp(t_k / T) / sum over the list, p_r = 0
 *   teacher_lse = l:      p_k = exp(t_k / T - l), p_r = max(0, 1 - sum p)   (l = log sum over ALL classes of exp(t / T);
 *                         p_r = 0 where the list holds every class)
 *   L = sum_k p_k (log p_k - log q_{i_k}) + p_r (log p_r - log sum_{v not in S} q_v)
 *   f = lam sum_n w_n L_n + label_lam sum_n w_n (log sum_v exp x_{n,v} - x_{n,y_n})     (y = -1: no label; labels may be NULL)
 * A class listed twice counts with both entries.  0 log 0 = 0.  A row of w = 0 is not read, its gradient is zero.  A row whose
 * scores are all -inf contributes nothing.  A listed class or a label at score -inf makes f = +inf where its mass is not zero,
 * and leaves the gradient finite.  A NaN among a row's scores, or an index or label outside [-1, classes), makes f and that
 * row's gradient NaN. */
typedef struct pg_distill {
  int64_t rows, classes, top; /* classes < 2^30, top <= 1024 */
  const void* teacher;        /* [rows x top], any element type; may be NULL with top = 0 */
  int64_t teacher_ld;
  const void* index; /* [rows x top], int32 or int64 */
  int64_t index_ld;
  const void* teacher_lse; /* [rows], PG_F32 or PG_F64; NULL: the list is renormalised */
  const void* weights;     /* [rows], PG_F32 or PG_F64; NULL: ones */
  const void* labels;      /* [rows], int32 or int64; NULL: none */
  int32_t teacher_dtype, index_bits, lse_dtype, weights_dtype, label_bits, reserved;
  double temperature, lam, label_lam; /* T > 0, lam >= 0, label_lam >= 0 */
} pg_distill;

pg_status pg_distill_value_and_gradient(pg_ctx* ctx, const pg_distill* d, int32_t dtype, const void* scores, int64_t ld,
                                        void* grad, int64_t grad_ld, void* value, double* f_out);

#ifdef __cplusplus
}
#endif
#endif /* PROXGRAD_HIP_ROWS_H */
