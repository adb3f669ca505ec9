/*
 * logits_process.h — C-ABI of the caption decoder's logits processing (csrc/logits_process.hip, built into
 * libmsda_hip.so): penalties for repeated tokens, biases and masks of allowed tokens, with the row's best token
 * and log-sum-exp, in one pass over the logits.
 *
 * Row i, token v, c = how often v is among tokens[i][0 .. token_lens[i]), in float32 and this order:
 *   x = logits[i][v]
 *   if c > 0:  x = x > 0 ? x / repetition : x * repetition;  x = x - presence;  x = x - frequency * c
 *   x = x + bias[i][v]
 *   x = -inf where the token is not allowed (whatever it was before)
 *   out[i][v] = x  (rounded to out's type),  best[i] = the lowest v of the largest x (NaN counts as the
 *   largest; -1 when every x is -inf),  lse[i] = log sum_v exp(x),  logprob[i] = -log sum_v exp(x - x[best])
 *   (-inf when best is -1, NaN when x[best] is infinite or NaN)
 *
 * logits (n, vocab) rows logits_row elements apart; dtype and out_dtype: 0 float32, 2 bfloat16, 3 float16.  out
 * may be logits itself (same type and stride), else must not overlap it; NULL: not written.  best / lse /
 * logprob may be NULL.  tokens (n, hist) int32, rows tokens_row apart; numbers outside [0, vocab) count nothing;
 * token_lens NULL: hist.  The penalties are per row where a pointer is given, else the scalar
 * (repetition: positive and finite in float32).  bias float32,
 * rows bias_row apart (0: one row).  allowed: allowed_kind 1 — bytes, non-zero = allowed; 2 — bits, token v
 * is bit v % 32 of int32 word v / 32; mask rows allowed_row bytes / words apart, allowed_rows of them; row i
 * takes mask row states[i] (outside [0, allowed_rows): everything is allowed), without states row i, or row 0
 * when allowed_rows is 1.  workspace: mfl_logits_workspace_bytes(args) bytes, 16-byte aligned.  Asynchronous
 * on `stream`, may be captured; 0, else non-zero with mfl_logits_last_error().
 */
#ifndef MFL_LOGITS_PROCESS_H
#define MFL_LOGITS_PROCESS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  const void* logits;
  void* out;
  int64_t* best;
  float *lse, *logprob;
  const int32_t *tokens, *token_lens;
  const float *repetition_rows, *presence_rows, *frequency_rows, *bias;
  const void* allowed;
  const int32_t* states;
  void* workspace;
  int64_t n, vocab, dtype, out_dtype, logits_row, out_row, hist, tokens_row, bias_row, allowed_kind, allowed_row,
      allowed_rows;
  double repetition, presence, frequency;
} mfl_logits_args;

int64_t mfl_logits_workspace_bytes(const mfl_logits_args* args);

int mfl_logits_process(const mfl_logits_args* args, void* stream);

const char* mfl_logits_last_error(void);

#ifdef __cplusplus
}
#endif

#endif
