/* zz_experts.h -- tokens to experts and back on the GPU (libzzmoe.so, MI355X gfx950): the
 * (token, slot) pairs of a routing in the experts' order with the tokens' rows, the way back
 * with the routing weights, and the gradients of both. For experts that zz_moe_forward (which
 * does all of this inside) does not hold: the 8-bit floating point tables of zz_fp8.h, or a
 * caller's own. The routing is what zz_moe_forward[_dev] gives as eidx and ewt, or any other.
 *
 * Conventions as zz_fp8.h: device pointers and a hipStream_t, no allocation, no wait,
 * capturable; 1 when done, 0 to decline with the outputs untouched.
 */
#ifndef ZZ_EXPERTS_H
#define ZZ_EXPERTS_H

#include <stdint.h>
#include <stddef.h>
#include "zz_fp8.h"

#define ZZ_EXPERTS_MAXE 512
#define ZZ_EXPERTS_MAXK 16

#ifdef __cplusplus
extern "C" {
#endif

/* Workspace of one zz_experts_dispatch_dev call of these sizes, in bytes; -1 for sizes that it
 * declines. The contents need no preparation and mean nothing afterwards. Calls that can
 * overlap (two streams, two graphs) take a workspace each. */
int64_t zz_experts_ws_bytes(int S, int K, int E);

/* The S x K pairs (s, j) of eidx [S][K] in the order of their experts, those of one expert in
 * their own order (the token, then the slot):
 *   offs [E + 1]   pairs of expert e are at the positions offs[e] .. offs[e + 1] - 1;
 *   pos [S][K]     the pair's position; -1 where eidx is outside 0 .. E-1: such a pair is
 *                  dropped, it has no position and no row;
 *   row [S * K]    the token at a position (position p's pair is (row[p], j) for the j with
 *                  pos[row[p]][j] = p); from offs[E] on left as it was.
 * and, where d_x is not NULL, the tokens' rows there: xs[pos[s][j]] = x[s], bit for bit. x [S, D]
 * and xs [S * K, D] are of `dtype`, rows ldx and ldxs elements apart (0: D); rows of xs from
 * offs[E] on, and what lies between rows, are left as they were. A token may name an expert
 * more than once. 1 <= S <= 2^20, 1 <= K <= 16, 1 <= E <= 512, 1 <= D <= 8192. Outputs overlap
 * nothing else (ranges are judged from their first byte to their last); d_ws is aligned to 4
 * bytes. */
int zz_experts_dispatch_dev(const int *d_eidx, int S, int K, int E, int *d_offs, int *d_row, int *d_pos,
                            int dtype, const void *d_x, int64_t ldx, int D, void *d_xs, int64_t ldxs,
                            void *d_ws, size_t ws_bytes, void *stream);

/* The way back: out[s] = res[s] + sum_j w[s][j] * y[pos[s][j]], j ascending, by one fma each in
 * f32, rounded once to `dtype`. A pair whose position is outside 0 .. S*K-1 adds nothing, its
 * weight unread. w [S][K] f32 (NULL: ones); res [S, D] (NULL: none) may be out itself, rows as
 * far apart. y [S * K, D], rows ldy apart (0: D; ldr, ldo likewise): only rows that pos names are
 * read. With w and res NULL this is the gradient of zz_experts_dispatch_dev's rows with respect
 * to x, y being the gradient of xs. The same sizes; out overlaps nothing else. */
int zz_experts_back_dev(int dtype, const void *d_y, int64_t ldy, const int *d_pos, const float *d_w, int S,
                        int K, int D, const void *d_res, int64_t ldr, void *d_out, int64_t ldo, void *stream);

/* The way back's gradient, dout [S, D] being that of out (and of res):
 *   dy[pos[s][j]] = w[s][j] * dout[s]            rounded once to `dtype`
 *   dw[s][j]      = sum_d dout[s][d] * y[pos[s][j]][d]     f32, 0 for a pair without a position
 * The sum over d is made of f32 sums of up to max(16, 8 ceil(D / 2048)) products each, joined in
 * pairs.
 * Rows of dy that pos does not name are left as they were; pos names a row once at most. dw
 * (NULL: not formed, y then unread and may be NULL); w NULL: ones. dout [S, D] rows ldg apart,
 * dy rows lddy. dy may be y itself, rows as far apart; outputs overlap nothing else. */
int zz_experts_back_grad_dev(int dtype, const void *d_dout, int64_t ldg, const void *d_y, int64_t ldy,
                             const int *d_pos, const float *d_w, int S, int K, int D, void *d_dy,
                             int64_t lddy, float *d_dw, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ZZ_EXPERTS_H */
