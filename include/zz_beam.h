/* zz_beam.h -- beam search's step on the GPU (libzzmoe.so, MI355X gfx950): selection over
 * beams and vocabulary, and the reordering of the beams' states. Beside the greedy
 * selection of zz_head_logits[_dev] (zz_gemma.h); zz_stack_beam_dev (zz_gemma.h) is a
 * stack's search with them. The reference decodes greedily or samples (gemma4.c:2147-2183)
 * and has no counterpart.
 *
 * Conventions as zz_fp8.h: device pointers, no allocation, no wait, capturable; 1 when
 * done, 0 to decline with the outputs untouched.
 */
#ifndef ZZ_BEAM_H
#define ZZ_BEAM_H

#include <stdint.h>
#include <stddef.h>
#include "zz_fp8.h"

#define ZZ_BEAM_MAXW 16
#define ZZ_BEAM_MAXV 524288

#ifdef __cplusplus
extern "C" {
#endif

/* Workspace of one zz_beam_step_dev call of these sizes, in bytes; -1 for sizes that it
 * declines. The contents need no preparation and mean nothing afterwards. Calls that can
 * overlap (two streams, two graphs) take a workspace each. */
int64_t zz_beam_ws_bytes(int N, int W, int V);

/* One step for N sequences of W beams (1 <= W <= 16, 1 <= V <= 524288, N * W <= 65535).
 * logits [N*W][V] of dtype, rows ldl elements apart (0: V); score [N][W] f32, the beams'
 * accumulated log-probabilities; done [N][W] bytes (NULL: none), nonzero for a finished
 * beam. A live beam w offers every token t at
 *   total = score[w] + logits[w][t] - log(sum_t' exp(logits[w][t']))
 * and a finished one offers `pad` alone at score[w], its logits unread. The W best of a
 * sequence are kept, in order: the larger total; equal totals, the lower beam, then the
 * larger logit, then the lower token. Totals are formed in double, from a logarithm whose sum
 * is made of f32's within 2048 or 8192 tokens and of doubles beyond: a total is off by up to
 * (2 ln V + 84) 2^-24 (6.5e-6 for 262144 tokens), and of two beams' totals that lie within
 * twice that either may come first. Within a beam the order is exact. A NaN logit counts as
 * minus infinity; a row whose largest logit is plus infinity shares its probability among
 * the infinite ones; a total that is NaN counts as minus infinity, which is a candidate
 * like others, so that W are always found.
 * Outputs [N][W]: score_out (f32), parent (the beam continued, 0 .. W-1), token,
 * done_out (NULL: not stored; 1 where the parent was finished or the token is `eos`; no
 * token is -1). score_out may be score and done_out may be done; nothing else overlaps.
 * d_ws is aligned to 8 bytes. */
int zz_beam_step_dev(int dtype, const void *d_logits, int64_t ldl, int N, int W, int V,
                     const float *d_score, const uint8_t *d_done, int eos, int pad, float *d_score_out,
                     int *d_parent, int *d_token, uint8_t *d_done_out, void *d_ws, size_t ws_bytes,
                     void *stream);

/* dst[o][n*W + w] = src[o][n*W + parent[n][w]] for o < outer, n < N, w < W: the first
 * row_bytes bytes of rows that lie row_stride bytes apart, in `outer` planes outer_stride
 * bytes apart (a cache of layers x rows x positions: the positions in use are moved, the
 * rest of a row is left as it was). dst is src itself (in place) or overlaps it nowhere;
 * row_bytes <= row_stride and N * W * row_stride <= outer_stride where outer > 1. A parent
 * outside 0 .. W-1 keeps the row. */
int zz_beam_reorder_dev(void *d_dst, const void *d_src, const int *d_parent, int N, int W, int64_t outer,
                        int64_t outer_stride, int64_t row_stride, int64_t row_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ZZ_BEAM_H */
