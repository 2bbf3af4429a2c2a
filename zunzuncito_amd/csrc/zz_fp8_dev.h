// zz_fp8_dev.h -- what the 8-bit floating-point kernels share (zz_fp8_rows.hip,
// zz_fp8_mma.hip) and their launchers.
#pragma once
#include "zz_common.h"

#define ZZ_F8B 128                  // elements under one scale
#define ZZ_F8MAX 448.0f             // largest e4m3 value
#define ZZ_F8FLOOR 0x1p-100f        // a block's largest magnitude counts as at least this

// element types of the unquantised side, as in include/zz_fp8.h
struct zz_bf16 { uint16_t u; };

__device__ __forceinline__ float zz_f32_of(float v) { return v; }
__device__ __forceinline__ float zz_f32_of(zz_bf16 v) { return __uint_as_float((unsigned)v.u << 16); }

// f32 -> bf16 bits, round to nearest even; a NaN stays one
__device__ __forceinline__ unsigned zz_bf16_bits(float f) {
    const unsigned u = __float_as_uint(f);
    const unsigned r = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
    return (u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : r;
}
__device__ __forceinline__ void zz_put(float *p, float v) { *p = v; }
__device__ __forceinline__ void zz_put(zz_bf16 *p, float v) { p->u = (uint16_t)zz_bf16_bits(v); }

// Four words at any address: rows of odd widths and strides begin at any multiple of their
// element, and the vector memory takes 16 bytes from there as well (by elements, a norm of 543 x
// 5035 bf16 rows took 21 us where it takes 9.5, a product of 6183 x 2889 x 176 34 where 22).
typedef unsigned zz_u4 __attribute__((ext_vector_type(4)));
typedef unsigned zz_u4any __attribute__((ext_vector_type(4), aligned(1), may_alias));
typedef unsigned zz_u2any __attribute__((ext_vector_type(2), aligned(1), may_alias));

// n (<= 8) consecutive elements as f32, zero behind them. over: 8 may be read all the same
template <typename T>
__device__ __forceinline__ void zz_get8(float (&v)[8], const T *p, int n, bool over) {
    if (n >= 8 || (over && n > 0)) {
        const zz_u4 a = *(const zz_u4any *)p;
        if constexpr (sizeof(T) == 4) {
            const zz_u4 b = *((const zz_u4any *)p + 1);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = __uint_as_float(a[j]);
                v[4 + j] = __uint_as_float(b[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] = __uint_as_float(a[j] << 16);
                v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
            }
        }
        if (n < 8)
#pragma unroll
            for (int j = 1; j < 8; j++) v[j] = j < n ? v[j] : 0.0f;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < n ? zz_f32_of(p[j]) : 0.0f;
}
// NT: stores that are not kept in the caches
template <bool NT, typename T>
__device__ __forceinline__ void zz_put8(T *p, const float (&v)[8], int n) {
    if (n >= 8) {
        zz_u4 w[sizeof(T) / 2];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j >> 2][j & 3] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) w[0][j] = zz_bf16_bits(v[2 * j]) | zz_bf16_bits(v[2 * j + 1]) << 16;
        }
#pragma unroll
        for (int j = 0; j < (int)(sizeof(T) / 2); j++) {
            if constexpr (NT) __builtin_nontemporal_store((zz_u4any)w[j], (zz_u4any *)p + j);
            else *((zz_u4any *)p + j) = w[j];
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < n) zz_put(p + j, v[j]);
}

// An output of at least this many bytes, a quarter of the 256 MB cache in front of memory, is
// stored past it: who reads it next finds little of it there, and its dirty lines would be
// written back under the next kernels' reads.
#define ZZ_NT_BYTES ((int64_t)64 << 20)

struct ZzF8RowsArgs {
    const void *x, *res;        // res, sum, w may be null
    void *sum;
    const float *w;
    int64_t ldx, ldr, lds;      // elements
    float eps;
    int S, D;
    int nt;                     // the sum is stored past the caches
    uint8_t *q;                 // [S][nb * 128]
    float *s;                   // [nb][S]
};
int zz_launch_add_norm_fp8(int dtype, const ZzF8RowsArgs &a, hipStream_t st);
int zz_launch_rows_fp8(int dtype, const ZzF8RowsArgs &a, hipStream_t st);

// A resident matrix: codes in 32-row groups, [O/32][nb][4][64 lanes][16 B], lane 32h + r of
// piece p holding row r's columns 32p + 16h .. + 15 of the block: what the lane's operands of
// the block's eight matrix-core steps are made of (step j: bytes 8 (j & 1) .. + 7 of piece
// j / 2). The steps' columns are in an order of their own, which the activation rows follow
// and a dot product does not see. Rows from O and columns from I on are zero.
struct ZzF8Mat {
    int O, I;
    const uint8_t *w;
    const float *ws;            // [ceil(O/128)][nb]
};
__host__ __device__ __forceinline__ int zz_f8_nb(int n) { return (n + ZZ_F8B - 1) / ZZ_F8B; }

int zz_launch_fp8_pack(const uint8_t *codes, int O, int I, uint8_t *dst, hipStream_t st);
int zz_launch_fp8_matmul(const ZzF8Mat &m, const uint8_t *q, const float *s, int S, int dtype, void *y,
                         int64_t ldy, hipStream_t st);
