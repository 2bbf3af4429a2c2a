/* zz_fp8.h -- rows and matrices of 8-bit floating point on the GPU (libzzmoe.so, MI355X
 * gfx950): the residual's addition, RMS norm and rounding of activation rows, and their
 * product with resident weights. For the dense projections around the MoE block whose
 * checkpoint is 8-bit floating point; beside gpu_matmul (zz_gpu.h), which takes the
 * integer formats.
 *
 * Values are e4m3 as OCP defines it (no infinities, 0x7F / 0xFF are NaN, largest 448).
 *   Rows [S, D]: codes, zz_fp8_row_bytes(D) bytes a row (D up to whole blocks of 128, the
 *     bytes from D on zero); scales f32 [ceil(D/128)][S], block-major: element d of row s
 *     is code[s][d] * scale[d/128][s].
 *   Matrices [O, I]: codes [O][I]; scales f32 [ceil(O/128)][ceil(I/128)], one for each
 *     128 x 128 block.
 *
 * Conventions as zz_moe.h: 1 when done, 0 (or -1 for an id) to decline with the outputs
 * untouched; single caller; _dev forms take device pointers and a hipStream_t (NULL = the
 * library's stream), allocate nothing, wait for nothing and can be captured into a graph.
 * They run on the device of gpu_init, which has to be the current one.
 */
#ifndef ZZ_FP8_H
#define ZZ_FP8_H

#include <stdint.h>
#include <stddef.h>
#include "zz_gpu.h"

/* element types of the unquantised side */
#define ZZ_F32  0
#define ZZ_BF16 1

/* activations of a product's epilogue */
#define ZZ_EP_NONE      0
#define ZZ_EP_GELU_TANH 1   /* v / (1 + exp(-sqrt(8/pi) (v + 0.044715 v^3))), gelu in its tanh form */
#define ZZ_EP_SILU      2   /* v / (1 + exp(-v)) */
/* or'ed to the activation: the caller takes sums of fewer bits for speed (zz_fp8_matmul_ep_dev) */
#define ZZ_EP_8BIT      16

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one row of D codes: D rounded up to a multiple of 128; -1 for D < 1. */
int64_t zz_fp8_row_bytes(int64_t D);

/* h = x + res (x where d_res is NULL), in f32; d_sum (NULL: not stored) receives h rounded
 * to dtype. y = h / sqrt(mean(h^2) + eps) * w, and each 128 of y as
 *   scale = max(max|y|, 2^-100) / 448,  code = e4m3(y / scale), round to nearest even,
 * both quotients those of f32, correctly rounded.
 * x, res and sum are of `dtype` with rows ldx, ldr, lds elements apart (0: D); w [D] is
 * f32 (NULL: ones). 1 <= D <= 8192, S <= 2^20. d_sum may be d_x or d_res itself, rows as
 * far apart; the outputs overlap nothing else (ranges are judged from their first byte to
 * their last, what lies between strided rows included). d_q is aligned to 16 bytes. The
 * squares, their mean and its root are in double, so that no row of finite h leaves their
 * range; a row of zeros with eps 0 is 0 / 0. A NaN or infinity in a row makes codes of that row NaN
 * or its scales infinite and touches no other row. */
int zz_add_norm_fp8_dev(int dtype, const void *d_x, int64_t ldx, const void *d_res, int64_t ldr,
                        void *d_sum, int64_t lds, const float *d_w, float eps, int S, int D,
                        uint8_t *d_q, float *d_s, void *stream);

/* The same rounding of x itself, without sum and norm: scales and codes are those of f32's
 * quotients to the last bit. Any D up to 2^20, S <= 2^24 (S * ceil(D/128) <= 2^27): the
 * rows that a table's product takes, too. */
int zz_rows_fp8_dev(int dtype, const void *d_x, int64_t ldx, int S, int D, uint8_t *d_q, float *d_s,
                    void *stream);

/* A resident matrix [O, I], O <= 2^24, I <= 65536, O * I < 2^35; returns its id, or -1.
 * Its weights are laid out once, in the matrix cores' order, by an upload (host or device
 * pointers; synchronous, on the library's stream: what fills d_codes and d_scales on another
 * stream, and calls with the matrix there, have to be waited for first). A later upload
 * replaces them. A matrix without an upload has no product; one that a captured graph uses
 * is destroyed after the graph. */
int zz_fp8_create(int O, int I);
void zz_fp8_destroy(int mat);
int zz_fp8_upload(int mat, const uint8_t *codes, const float *scales);
int zz_fp8_upload_dev(int mat, const uint8_t *d_codes, const float *d_scales);

/* y [S, O] = rows [S, I] times the matrix's transpose: for each block of 128 columns the
 * codes' product in f32, times the f32 product of the row's and the block's scale, added up
 * in f32 in the order of the columns or of groups of them; rounded once to `dtype`. Rows of
 * y are ldy elements apart (0: O); what lies between them is left as it was. S <= 2^20,
 * S * O < 2^37. d_q is aligned to 16 bytes. Results do not depend on other rows' values and
 * are the same on every call of the same sizes. */
int zz_fp8_matmul_dev(int mat, const uint8_t *d_q, const float *d_s, int S, int dtype, void *d_y,
                      int64_t ldy, void *stream);

/* Host form, synchronous: x [S, I] f32 is rounded as zz_rows_fp8_dev does and multiplied;
 * y [S, O] f32. */
int zz_fp8_matmul(int mat, const float *x, float *y, int S);

/* A resident table of E experts' matrices [O, I] (E = 1: one matrix), or with `gated` of E pairs
 * of them, gate and up; returns its id, or -1. zz_fp8_destroy gives it back. 1 <= E <= 512, O
 * and I as zz_fp8_create's, all codes together less than 2^38 bytes. An upload fills one matrix,
 * part 0 the only or the gate's, part 1 the up's, codes and scales as zz_fp8_upload's, and under
 * its conditions; a table whose uploads are not complete has no product. */
int zz_fp8_create_experts(int E, int O, int I, int gated);
int zz_fp8_upload_expert(int mat, int e, int part, const uint8_t *codes, const float *scales);
int zz_fp8_upload_expert_dev(int mat, int e, int part, const uint8_t *d_codes, const float *d_scales);

/* The product of one matrix (zz_fp8_create's, or a table's with E = 1) with an epilogue: v the
 * sums of zz_fp8_matmul_dev (not rounded) plus bias, then
 *   y = act(v) + res                                        a plain matrix
 *   y = act(min(v_gate, clamp)) * clip(v_up, -clamp, clamp) + res       a gated pair
 * in f32, rounded once to `dtype`. bias f32 [O], a gated pair's [2][O], gate's first (NULL:
 * none); act ZZ_EP_*, with or without ZZ_EP_8BIT; clamp > 0, or 0 for none (a plain matrix takes
 * none); res [S, O] of `dtype`, rows ldr apart (0: O; NULL: none), may be y itself, rows as far apart. The
 * activations are of one hardware exponential and one reciprocal: off by up to (6 + 10 |a|) 2^-24 of
 * the value, a the exponent, beside what v is off; where a is above 87.3, so that 1 / (1 + exp(a)) is less than
 * 2^-126, they may be 0 for less than |v| 2^-126. A NaN stays one; act(-infinity) is NaN, infinity
 * times 0. The order in which the blocks of 128 columns are added up follows from the sizes, S among them:
 * a row's result can differ in its last bits between calls of different S.
 * With ZZ_EP_8BIT in act, results in bf16 of more than some dozens of rows come from the 8-bit matrix
 * instructions, at up to twice the rate: within each 8 columns a product is cut, towards zero, to 13
 * bits behind the leading one of the largest, before they are added up in f32. That is 1.4e-5 of the
 * 2-norm for normally distributed codes and less than 8.6e-4 of the terms' magnitudes at worst, beside
 * the 2^-8 of a result's rounding; where terms cancel, of the result it can be any part. Results in
 * f32 and of few rows are the same with it and without. Other limits and promises as
 * zz_fp8_matmul_dev's, S <= 2^20, and results are of less than 2^24 tiles of 128 rows and 128 columns (a
 * gated pair's: 64). y overlaps no other argument. */
int zz_fp8_matmul_ep_dev(int mat, const uint8_t *d_q, const float *d_s, int S, const float *d_bias, int act,
                         float clamp, const void *d_res, int64_t ldr, int dtype, void *d_y, int64_t ldy,
                         void *stream);

/* The same over a table of experts: rows offs[e] .. offs[e + 1] - 1 of y [P, O] are expert e's
 * products, of the rows row[p] of the R rows in d_q, d_s (row NULL: of row p itself, R >= P).
 * offs [E + 1] and row [P] are device memory (zz_experts_dispatch_dev makes them): offs ascends from
 * 0 or more to P or less, rows of y outside it are left as they were; with an index outside 0 ..
 * R-1 row 0 is taken. bias [E][O], gated [E][2][O]; res [P, O]. P, R <= 2^24; with d_row, R *
 * zz_fp8_row_bytes(I) < 2^32. Tiles count as (P + 127 min(E, P)) / 128 of rows times those of columns. The
 * form is chosen by the table's size and P: rows' results do not depend on how many rows other experts
 * have. With ZZ_EP_8BIT a table's results in bf16 can come from the 8-bit instructions however few rows
 * an expert has. */
int zz_fp8_matmul_experts_dev(int mat, const uint8_t *d_q, const float *d_s, int R, const int *d_row,
                              const int *d_offs, int P, const float *d_bias, int act, float clamp,
                              const void *d_res, int64_t ldr, int dtype, void *d_y, int64_t ldy, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ZZ_FP8_H */
