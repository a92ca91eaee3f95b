/*
 * C ABI of beam search's selection in libl20_paged_decode_hip.so: the best continuations of each request's
 * beams over the vocabulary.  Return codes and l20_pd_last_error() are those of l20_paged_decode.h.  The
 * reference decodes greedily or by verification: no counterpart there.
 */
#ifndef L20_BEAM_SEARCH_H_
#define L20_BEAM_SEARCH_H_

#include <stdint.h>

#include "l20_paged_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

#define L20_PD_MAX_BEAMS 32
#define L20_PD_MAX_END_TOKENS 8

/*
 * One step of `requests` searches of `beams` beams.  Strides are in elements; the vocabulary is contiguous.
 *
 *   logits  [requests, beams, vocab] dtype (bf16, fp16 or fp32), rows of any alignment of the element
 *   scores  [requests, beams] fp32, the beams' summed log-probabilities; a beam whose score is not finite
 *           is dead: its logits do not matter
 *   end_tokens  HOST array of num_end_tokens ids
 *
 * The candidate (w, v) of a request has the score  s = scores[w] + (logits[w][v] - log sum_u exp logits[w][u])
 * and counts if s is finite in 32 bits: a row that holds a NaN or +inf, or -inf alone, has no candidates, and
 * neither has a token of -inf.  Candidates are ordered by s (in 64 bits, falling), then by beam (rising), by
 * logit (falling) and by token (rising).
 *
 *   tokens, parents, scores_out     [requests, beams] contiguous: the first `beams` candidates whose token is
 *                                   no end token; -1, -1 and -inf where there are fewer.  scores_out may be
 *                                   scores itself
 *   ended_tokens, _parents, _scores the candidates with an end token among the first `beams` of all, in
 *                                   order; -1, -1 and -inf behind them
 *
 * Two launches, nothing allocated.  Atomics are on whole numbers, whose order does not matter: equal inputs give equal
 * bits.  The workspace's contents do not matter; calls that may overlap each need their own.
 */
typedef struct l20_pd_beam_step_args {
  const void *logits;
  int64_t l_stride_request, l_stride_beam;
  int32_t dtype;
  const float *scores;
  int64_t s_stride_request, s_stride_beam;
  int32_t requests, beams, vocab;
  const int32_t *end_tokens;
  int32_t num_end_tokens;
  int64_t *tokens;
  int32_t *parents;
  float *scores_out;
  int64_t *ended_tokens;
  int32_t *ended_parents;
  float *ended_scores;
  void *workspace;
  int64_t workspace_bytes;
} l20_pd_beam_step_args;

int32_t l20_pd_beam_step_check(const l20_pd_beam_step_args *args);

/* Bytes of workspace for these requests, beams, vocab and num_end_tokens (and for any fewer of each). */
int64_t l20_pd_beam_step_workspace(const l20_pd_beam_step_args *args);

int32_t l20_pd_beam_step(const l20_pd_beam_step_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* L20_BEAM_SEARCH_H_ */
