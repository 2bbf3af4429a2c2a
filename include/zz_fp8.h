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
 * quotients to the last bit. Any D up to 2^20, S <= 2^20 (S * ceil(D/128) <= 2^27). */
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

#ifdef __cplusplus
}
#endif

#endif /* ZZ_FP8_H */
