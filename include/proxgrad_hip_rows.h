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
 * rounded to the scores' type once.  In Float32 a probability of less than 2^-97 of the row's largest may be 0.
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
 * scores are all -inf contributes nothing.  A listed class, a label or all that is outside the list at score -inf makes f = +inf
 * where its mass and its factor (lam, label_lam) are not zero, and leaves the gradient finite.  A NaN among a row's scores, or an index or label outside [-1, classes), makes f and that
 * row's gradient NaN. */
typedef struct pg_distill {
  int64_t rows, classes, top; /* classes <= 2^24, top <= 1024 */
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

/* ------------------------------------------------------------------ balance of a router's experts ---- */
/* Scores r (tokens x experts), p = softmax(r) of a token; tokens in groups g (all of them one group, or one per sequence), mask:
 *   c_ge = how often the group's unmasked tokens choose expert e,  n_g = number of its unmasked tokens
 *   f = lam sum_g experts / (k n_g^2) sum_e c_ge sum_{t in g} p_te          (lam per group at perfect balance)
 *   df/dr_tj = a_g p_tj (c_gj - sum_e c_ge p_te),  a_g = lam experts / (k n_g^2)      (the counts held fixed)
 * chosen == NULL: a token chooses its k highest scores, the lowest index first among equal ones; -inf and NaN are never chosen.
 * chosen: the router's own choices [tokens x k], -1 = none; an expert named twice counts twice.
 * A masked token counts for nothing, whatever its scores and choices hold, and its gradient is zero.  A token whose scores are all -inf has gradient zero.
 * A NaN among a token's scores makes f and that token's gradient NaN; a choice outside [-1, experts) makes f and its
 * group's gradients NaN.  A group without unmasked tokens contributes nothing.  The tiles say what is read and written:
 * tokens of a tile of group -1 belong to no group and get a zero gradient, tokens of no tile are left alone. */
typedef struct pg_balance_tile {
  int64_t begin, end; /* tokens [begin, end) of one group */
  int32_t group;      /* -1: tokens of no group */
  int32_t part; /* its number within the group; -1: the group's only tile */
} pg_balance_tile;
typedef struct pg_balance {
  int64_t tokens, groups, ntiles; /* tokens < 2^31 */
  int64_t tile_tokens;            /* tiles == NULL: one group of all tokens, in tiles of this many (the last one shorter) */
  const pg_balance_tile* tiles;   /* device; every token in at most one tile, a group's tiles in any order */
  const void* mask;               /* [tokens] bytes, 0 = masked; NULL: none */
  const void* chosen;             /* [tokens x k] int32 or int64; NULL: the k highest */
  int64_t chosen_ld;
  int32_t* counts;  /* device [groups x experts]: c of the last evaluation (groups without tiles are left alone) */
  uint32_t* state;  /* device, 4 + 2 * groups * copies * (experts + 2) words, zero before the first evaluation: this loss's own */
  int32_t experts, k, chosen_bits; /* 1 <= k <= experts <= 1024 */
  int32_t whole;                   /* every tile is a whole group: one launch (state: 4 words) */
  int32_t copies, reserved;        /* accumulators per group that its tiles take in turn, 1 .. 16 */
  double lam;
} pg_balance;

pg_status pg_balance_value_and_gradient(pg_ctx* ctx, const pg_balance* b, int32_t dtype, const void* scores, int64_t ld,
                                        void* grad, int64_t grad_ld, void* value, double* f_out);

#ifdef __cplusplus
}
#endif
#endif /* PROXGRAD_HIP_ROWS_H */
