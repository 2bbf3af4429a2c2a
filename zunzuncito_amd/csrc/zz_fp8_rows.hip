// zz_fp8_rows.hip -- activation rows to e4m3 codes with an f32 scale per 128 elements
// (include/zz_fp8.h), with the residual's addition and the RMS norm before it or without.
//
//   h = x + res;  r = 1 / sqrt(sum(h^2) / D + eps);  y = (h * r) * w
// The squares, their sum and r are in double: no row's leave its range, and beside the row's bytes
// they cost nothing (58.4 us and 58.0 at 8192 x 2816). r is rounded to f32 for the product with h,
// which is formed in double for the rows whose r has no place there (in double for all, with w
// too, 8192 x 2816 in bf16 took 43 us for 41).
//   per 128: a = max(max|y|, 2^-100), scale = a / 448, code = e4m3(y / scale)
// Both quotients are f32's, correctly rounded: values of few bits, as bf16 rows are, often lie
// right between two codes, where the last bit of y / scale decides for a whole step (with
// y * (448 / a) 3e-4 of such rows' codes are a neighbour of the right one; 1500 x 2112 bf16 took
// 4.1 us with that and take 4.3). |y| <= a keeps y / scale under 448 * (1 + 2^-22), which rounds
// to 448.
//
// A thread holds 8 consecutive elements: 16 lanes are one block, so its maximum is four DPP
// steps and a code group one 8-byte store.
#include "zz_fp8_dev.h"

// 16 lanes' 8 values each -> their codes (two words) and the block's scale
__device__ __forceinline__ uint2 zz_f8_block(const float (&y)[8], float *scale) {
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) a = fmaxf(a, fabsf(y[j]));
    a = fmaxf(zz_group_max<16>(a), ZZ_F8FLOOR);
    // a / 448, rounded right by one step: no quotient by 7 comes near the middle between two floats
    constexpr float c448 = 1.0f / ZZ_F8MAX;
    const float s0 = a * c448, s = a < INFINITY ? fmaf(-fmaf(s0, ZZ_F8MAX, -a), c448, s0) : a;
    *scale = s;
    // y / s by the block's one reciprocal: t is at most 1.5 ulp off, and what one step with its
    // remainder leaves, 2^-22 ulp, could only change a code where y / s lies that near to the
    // middle between one of the codes' borders (five bits) and its neighbour. Those pairs, with s
    // within 2^-20 of four bits, were all looked at: each rounds as the division does. Blocks
    // whose remainders could be subnormal are made larger first; under an infinite scale what is
    // finite is 0.
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = y[j];
    float d = s;
    if (a < 0x1p-80f) {
        d *= 0x1p64f;
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] *= 0x1p64f;
    }
    const float inv = 1.0f / d;
    d = a < INFINITY ? d : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float t = q[j] * inv;
        q[j] = fmaf(-fmaf(t, d, -q[j]), inv, t);         // (a zero keeps its sign)
    }
    int c[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k], q[4 * k + 1], 0, false);
        c[k] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k + 2], q[4 * k + 3], w, true);
    }
    return make_uint2((unsigned)c[0], (unsigned)c[1]);
}

// 8192 x 2816 in f32 take 58.5 us, 5.1 TB/s, which is what a large copy reaches (63 with the sum
// kept in the caches), in bf16 41; one row 3.5 us, a launch's 2.2 and one trip to memory.
// TPR threads per row, NU groups of 8 per thread held in registers between the sum of squares
// and the codes: x and res are read once, sum and codes written once. As few threads as hold a
// row with one group each, at least a wave: 6000 x 512 bf16 rows take 6.9 us with a wave each
// and 11.8 with four, 6000 x 1024 10.9 with two and 13.3 with four; with fewer threads and two
// groups each a single row takes longer (1024: 3.4 for 2.7).
// In 16 bits a row's last group, where 8 do not divide the width, reads on into the next row,
// which the last row has not (6000 x 742: 11.4 us for 14.5; in f32 it lost, 13.7 for 13.0).
template <typename T, int TPR, int NU, bool NT>
__global__ __launch_bounds__(256) void zz_add_norm_fp8_kernel(ZzF8RowsArgs a) {
    __shared__ double red[4];
    const int tid = threadIdx.x % TPR, D = a.D, nb = zz_f8_nb(D);
    const int own = TPR == 256 ? blockIdx.x : blockIdx.x * (256 / TPR) + threadIdx.x / TPR, row = min(own, a.S - 1);
    const bool over = sizeof(T) == 2 && row < a.S - 1 && D >= 8;
    const T *x = (const T *)a.x + row * a.ldx;
    const T *res = a.res ? (const T *)a.res + row * a.ldr : nullptr;
    T *sum = a.sum ? (T *)a.sum + row * a.lds : nullptr;
    float h[NU][8];
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int e = 8 * (i * TPR + tid);
        zz_get8(h[i], x + e, D - e, over);
        if (res) {
            float t[8];
            zz_get8(t, res + e, D - e, over);
#pragma unroll
            for (int j = 0; j < 8; j++) h[i][j] += t[j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fma((double)h[i][j], (double)h[i][j], ss);
        if (sum && e < D && own < a.S) zz_put8<NT>(sum + e, h[i], D - e);
    }
    double t = zz_wave_sum(ss);
    if constexpr (TPR > 64) {
        constexpr int RW = TPR / 64;                      // a row's waves
        const int wave = threadIdx.x >> 6, first = wave / RW * RW;
        if ((tid & 63) == 0) red[wave] = t;
        __syncthreads();
        t = RW == 4 ? (red[0] + red[1]) + (red[2] + red[3]) : red[first] + red[first + 1];
    }
    if (own >= a.S) return;
    const double rd = 1.0 / sqrt(t / D + (double)a.eps);
    float r = (float)rd;
    if (!(rd >= 0x1p-126 && rd <= 0x1p126)) {              // f32 does not hold it with all its bits
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                asm volatile("" : "+v"(h[i][j]));         // the squares' doubles are not kept for here
                h[i][j] = (float)((double)h[i][j] * rd);
            }
        r = 1.0f;
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int e = 8 * (i * TPR + tid);
        float w[8];
        if (a.w) {
            zz_get8(w, a.w + e, D - e, false);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = 1.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = (h[i][j] * r) * w[j];
        float sc;
        const uint2 c = zz_f8_block(h[i], &sc);
        if (e < nb * ZZ_F8B) {
            *(uint2 *)(a.q + (size_t)row * nb * ZZ_F8B + e) = c;
            if ((tid & 15) == 0) a.s[(size_t)(e / ZZ_F8B) * a.S + row] = sc;
        }
    }
}

// Blocks of rows without a norm: 16 lanes per block, 16 blocks per workgroup.
template <typename T>
__global__ __launch_bounds__(256) void zz_rows_fp8_kernel(ZzF8RowsArgs a) {
    const int nb = zz_f8_nb(a.D), total = a.S * nb;
    const int id = blockIdx.x * 16 + (threadIdx.x >> 4), m = threadIdx.x & 15;
    const int at = id < total ? id : total - 1, row = at / nb, b = at - row * nb;
    const int e = b * ZZ_F8B + 8 * m;
    float v[8];
    zz_get8(v, (const T *)a.x + row * a.ldx + e, a.D - e, sizeof(T) == 2 && row < a.S - 1 && a.D >= 8);
    float sc;
    const uint2 c = zz_f8_block(v, &sc);
    if (id >= total) return;
    *(uint2 *)(a.q + (size_t)row * nb * ZZ_F8B + e) = c;
    if (m == 0) a.s[(size_t)b * a.S + row] = sc;
}

template <typename T, int TPR, int NU, bool NT>
static void launch_norm(const ZzF8RowsArgs &a, hipStream_t st) {
    hipLaunchKernelGGL((zz_add_norm_fp8_kernel<T, TPR, NU, NT>), dim3((a.S + 256 / TPR - 1) / (256 / TPR)), dim3(256), 0, st, a);
}
template <typename T, bool NT>
static void launch_norm(const ZzF8RowsArgs &a, hipStream_t st) {
    const int lanes = zz_f8_nb(a.D) * 16;
    if (lanes <= 64) launch_norm<T, 64, 1, NT>(a, st);
    else if (lanes <= 128) launch_norm<T, 128, 1, NT>(a, st);
    else if (lanes <= 256) launch_norm<T, 256, 1, NT>(a, st);
    else if (lanes <= 512) launch_norm<T, 256, 2, NT>(a, st);
    else launch_norm<T, 256, 4, NT>(a, st);
}

int zz_launch_add_norm_fp8(int dtype, const ZzF8RowsArgs &a, hipStream_t st) {
    if (dtype == 0) a.nt ? launch_norm<float, true>(a, st) : launch_norm<float, false>(a, st);
    else a.nt ? launch_norm<zz_bf16, true>(a, st) : launch_norm<zz_bf16, false>(a, st);
    return hipGetLastError() == hipSuccess;
}

int zz_launch_rows_fp8(int dtype, const ZzF8RowsArgs &a, hipStream_t st) {
    const dim3 g((unsigned)(((int64_t)a.S * zz_f8_nb(a.D) + 15) / 16)), b(256);
    if (dtype == 0) hipLaunchKernelGGL((zz_rows_fp8_kernel<float>), g, b, 0, st, a);
    else hipLaunchKernelGGL((zz_rows_fp8_kernel<zz_bf16>), g, b, 0, st, a);
    return hipGetLastError() == hipSuccess;
}
