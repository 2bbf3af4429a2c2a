// zz_fp8_mma.hip -- products of e4m3 rows with resident e4m3 matrices on the matrix cores
// (include/zz_fp8.h).
//
//   y[s][o] = sum_b xs[b][s] * ws[o/128][b] * sum_{k in block b} xq[s][k] wq[o][k]
// The codes are multiplied as f16, which holds every e4m3 value: the products are exact and
// the matrix core adds them up in f32. The 8-bit instructions do not: they align 16 products
// to the largest and keep 13 bits behind it (2^-14 beside 1 is lost within 16 neighbours and
// kept between them, measured), 1.5e-5 off in the 2-norm over normally distributed codes and
// 1e-4 of the terms' magnitude at worst, where the f16 form is 1e-8 and 2e-7 off. They would
// run at twice the rate.
//
// A block of 128 columns is four v_mfma_f32_16x16x32_f16 of 16 matrix rows times 16
// activation rows; each of the four results a lane then enters the f32 accumulator by one
// fma with the two scales' product. Lane 16q + r of a result holds matrix rows 4q..4q+3 of
// the group and activation row r, so a lane needs one row scale and a group one matrix scale.
#include "zz_fp8_dev.h"

typedef _Float16 zz_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 zz_h8 __attribute__((ext_vector_type(8)));
typedef float zz_v4f __attribute__((ext_vector_type(4)));

// 8 codes (two words) as f16: v_cvt_scalef32_pk_f16_fp8 at scale 1, exact, NaN stays NaN
__device__ __forceinline__ zz_h8 zz_f8_half(unsigned a, unsigned b) {
    const zz_h2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, false);
    const zz_h2 q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, true);
    const zz_h2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, false);
    const zz_h2 t = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, true);
    return zz_h8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
}

// the four steps' operands of a lane's two 16-byte pieces of a block
struct ZzF8Frag { zz_h8 h[4]; };
__device__ __forceinline__ ZzF8Frag zz_f8_frag(uint4 a, uint4 b) {
    return {{zz_f8_half(a.x, a.y), zz_f8_half(a.z, a.w), zz_f8_half(b.x, b.y), zz_f8_half(b.z, b.w)}};
}
__device__ __forceinline__ zz_v4f zz_f8_mma(const ZzF8Frag &a, const ZzF8Frag &b) {
    zz_v4f c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h[j], b.h[j], c, 0, 0, 0);
    return c;
}

// matrix rows o..o+3 of activation row t
template <typename T>
__device__ __forceinline__ void zz_f8_store4(T *y, int64_t ldy, int t, int o, int O, bool vec, const float (&v)[4]) {
    T *p = y + (int64_t)t * ldy + o;
    if (vec && o + 4 <= O) {
        if constexpr (sizeof(T) == 4) *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
        else *(uint2 *)p = make_uint2(zz_bf16_bits(v[0]) | zz_bf16_bits(v[1]) << 16,
                                      zz_bf16_bits(v[2]) | zz_bf16_bits(v[3]) << 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (o + i < O) zz_put(p + i, v[i]);
}

struct ZzF8Mm {
    ZzF8Mat m;
    const uint8_t *q;
    const float *s;
    int S, nb, vec;
    void *y;
    int64_t ldy;
};

// One workgroup per 16 matrix rows and 16 activation rows; its waves take every fourth
// block and meet in LDS, where the partial sums are added in the waves' order. Rows behind
// the last one are read as the last one, and not stored.
template <typename T>
__global__ __launch_bounds__(256) void zz_fp8_mm_kernel(ZzF8Mm a) {
    __shared__ float part[4][64][4];
    const int tid = threadIdx.x, w = zz_wave_id(), l = tid & 63, r = l & 15, qq = l >> 4;
    const int g = blockIdx.x, t = blockIdx.y * 16 + r, tc = min(t, a.S - 1), nb = a.nb;
    const uint8_t *wp = a.m.w + (size_t)g * nb * 2048 + l * 16;
    const uint8_t *xp = a.q + (size_t)tc * nb * ZZ_F8B + 16 * qq;
    const float *ws = a.m.ws + (size_t)(g / 8) * nb;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = w; b < nb; b += 4) {
        const uint4 w0 = *(const uint4 *)(wp + (size_t)b * 2048), w1 = *(const uint4 *)(wp + (size_t)b * 2048 + 1024);
        const uint4 x0 = *(const uint4 *)(xp + b * ZZ_F8B), x1 = *(const uint4 *)(xp + b * ZZ_F8B + 64);
        const float sc = a.s[(size_t)b * a.S + tc] * ws[b];
        const zz_v4f p = zz_f8_mma(zz_f8_frag(w0, w1), zz_f8_frag(x0, x1));
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(p[i], sc, acc[i]);
    }
    *(float4 *)part[w][l] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (w == 0 && t < a.S) {
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = (part[0][l][i] + part[1][l][i]) + (part[2][l][i] + part[3][l][i]);
        zz_f8_store4((T *)a.y, a.ldy, t, 16 * g + 4 * qq, a.m.O, a.vec, acc);
    }
}

// one 16-byte piece of the packed layout per thread
__global__ __launch_bounds__(256) void zz_fp8_pack_kernel(const uint8_t *src, int O, int I, int nb, uint8_t *dst,
                                                          int64_t n) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    const int l = (int)(p & 63), h = (int)(p >> 6) & 1;
    const int64_t gb = p >> 7, g = gb / nb;
    const int b = (int)(gb - g * nb), k = b * ZZ_F8B + 64 * h + 16 * (l >> 4);
    const int64_t row = g * 16 + (l & 15);
    unsigned w[4] = {0, 0, 0, 0};
    if (row < O) {
        const uint8_t *s = src + row * I + k;
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (k + j < I) w[j >> 2] |= (unsigned)s[j] << (8 * (j & 3));
    }
    *(uint4 *)(dst + 16 * p) = make_uint4(w[0], w[1], w[2], w[3]);
}

int zz_launch_fp8_pack(const uint8_t *codes, int O, int I, uint8_t *dst, hipStream_t st) {
    const int nb = zz_f8_nb(I);
    const int64_t n = (int64_t)((O + 15) / 16) * nb * 128;
    hipLaunchKernelGGL(zz_fp8_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, codes, O, I, nb, dst, n);
    return hipGetLastError() == hipSuccess;
}

template <typename T>
static void launch_mm(const ZzF8Mm &a, hipStream_t st) {
    hipLaunchKernelGGL(zz_fp8_mm_kernel<T>, dim3((a.m.O + 15) / 16, (a.S + 15) / 16), dim3(256), 0, st, a);
}

int zz_launch_fp8_matmul(const ZzF8Mat &m, const uint8_t *q, const float *s, int S, int dtype, void *y,
                         int64_t ldy, hipStream_t st) {
    const int esz = dtype == 0 ? 4 : 2;
    ZzF8Mm a{m, q, s, S, zz_f8_nb(m.I), 0, y, ldy};
    a.vec = (uintptr_t)y % (4 * esz) == 0 && ldy % 4 == 0;
    dtype == 0 ? launch_mm<float>(a, st) : launch_mm<zz_bf16>(a, st);
    return hipGetLastError() == hipSuccess;
}
