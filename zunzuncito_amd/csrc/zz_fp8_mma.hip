// zz_fp8_mma.hip -- products of e4m3 rows with one plain resident matrix (include/zz_fp8.h): the
// kernels, which form a call takes, and the codes' layout.
#include "zz_fp8_mma.h"

template <typename T, int RG, int RS, int NW, bool PF, bool NT>
__global__ __launch_bounds__(64 * NW) void zz_fp8_few_kernel(ZzF8Mm a) {
    extern __shared__ __attribute__((aligned(16))) float part[];
    zz_fp8_few<T, 0, RG, RS, NW, PF, NT>(a, part, blockIdx.x * RG, blockIdx.y * 32 * RS);
}

template <typename T, int RO, int RS, int WO, int WS, int KS, int NS>
__global__ __launch_bounds__(64 * WO * WS * KS, 2) void zz_fp8_async_kernel(ZzF8Mm a) {
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int OT = (a.m.O + C::O - 1) / C::O, ST = (a.S + C::S - 1) / C::S;
    const int id = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    if (id >= OT * ST) return;
    int ot, st;
    zz_fp8_at(id, OT, ST, &ot, &st);
    zz_fp8_tile<T, 0, RO, RS, WO, WS, KS, NS, false>(a, lds, ot * C::O / 32, st * C::S);
}

// Tiles of 64 RO x 64 RS; those from `whole` on in parts of 64 x 64, which run as a last round
// of their own or beside a last round of whole tiles.
template <typename T, int RO, int RS, bool NT>
__global__ __launch_bounds__(256, 2) void zz_fp8_tiles_kernel(ZzF8Mm a, int whole) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int OT = (a.m.O + 64 * RO - 1) / (64 * RO), ST = (a.S + 64 * RS - 1) / (64 * RS);
    const int g = (whole + 7) / 8, x = blockIdx.x;
    int ot, st;
    if (x < 8 * g) {
        const int id = x % 8 * g + x / 8;
        if (id >= whole) return;
        zz_fp8_at(id, OT, ST, &ot, &st);
        zz_fp8_tile<T, 0, RO, RS, 2, 2, 1, 2, NT>(a, lds, ot * 2 * RO, st * 64 * RS);
    } else {
        const int part = (x - 8 * g) % (RO * RS);
        zz_fp8_at(whole + (x - 8 * g) / (RO * RS), OT, ST, &ot, &st);
        const int gt = (ot * RO + part % RO) * 2, t0 = (st * RS + part / RO) * 64;
        if (gt * 32 < a.m.O && t0 < a.S) zz_fp8_tile<T, 0, 1, 1, 2, 2, 1, 3, NT>(a, lds, gt, t0);
    }
}

// one 16-byte piece of the packed layout per thread; part 0, 1: gate's, up's rows of a gated pair
// (-1: a plain matrix), the other's left as they are. The first threads copy the scales, of which
// there are fewer than pieces.
__global__ __launch_bounds__(256) void zz_fp8_pack_kernel(const uint8_t *src, int O, int I, int nb, uint8_t *dst,
                                                          int64_t n, int part, const float *scales, float *ws, int ns) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p < ns) ws[p] = scales[p];
    if (p >= n) return;
    const int l = (int)(p & 63), pc = (int)(p >> 6) & 3;
    const int64_t gb = p >> 8, g = gb / nb;
    const int b = (int)(gb - g * nb), k = b * ZZ_F8B + 32 * pc + 16 * (l >> 5);
    int64_t row = g * 32 + (l & 31);
    if (part >= 0) {
        if (((l >> 4) & 1) != part) return;
        row = g * 16 + (l & 15);
    }
    unsigned w[4] = {0, 0, 0, 0};
    if (row < O) {
        const uint8_t *s = src + row * I + k;
        if (k + 16 <= I) {
            __builtin_memcpy(w, s, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (k + j < I) w[j >> 2] |= (unsigned)s[j] << (8 * (j & 3));
        }
    }
    *(uint4 *)(dst + 16 * p) = make_uint4(w[0], w[1], w[2], w[3]);
}

int zz_launch_fp8_pack(const uint8_t *codes, int O, int I, int part, uint8_t *dst, const float *scales, float *ws, hipStream_t st) {
    const int nb = zz_f8_nb(I), gc = part < 0 ? 32 : 16;
    const int64_t n = (int64_t)((O + gc - 1) / gc) * nb * 256;
    hipLaunchKernelGGL(zz_fp8_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, codes, O, I, nb, dst, n, part,
                       scales, ws, scales ? zz_f8_nb(O) * nb : 0);
    return hipGetLastError() == hipSuccess;
}

template <typename T, int RO, int RS, int WO, int WS, int KS, int NS>
static bool launch_async(const ZzF8Mm &a, hipStream_t st) {
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    const int64_t n = ((int64_t)((a.m.O + C::O - 1) / C::O) * ((a.S + C::S - 1) / C::S) + 7) / 8 * 8;
    if (n * C::NT > 0xffffffffll) return false;           // a launch's threads in one dimension
    hipLaunchKernelGGL((zz_fp8_async_kernel<T, RO, RS, WO, WS, KS, NS>), dim3((unsigned)n), dim3(C::NT), C::LDS, st, a);
    return true;
}

template <typename T, int RO, int RS>
static bool launch_tiles(const ZzF8Mm &a, bool split, hipStream_t st) {
    typedef ZzF8Async<RO, RS, 2, 2, 1, 2> C;
    typedef ZzF8Async<1, 1, 2, 2, 1, 3> P;
    const int64_t n = (int64_t)((a.m.O + C::O - 1) / C::O) * ((a.S + C::S - 1) / C::S);
    const int64_t whole = split ? n - n % 256 : n, g = (whole + 7) / 8 * 8 + (n - whole) * RO * RS;
    if (g * C::NT > 0xffffffffll) return false;           // a launch's threads in one dimension
    // large results past the caches (4096 x 8192 x 256 in f32 53 us and 38), where tiles write
    // whole lines; else every line is written twice (8192 x 2892 x 256 in f32 33 us and 43)
    const bool nt = a.S * a.ldy * (int64_t)sizeof(T) >= ZZ_NT_BYTES &&
                    (uintptr_t)a.y % 64 == 0 && a.ldy * sizeof(T) % 64 == 0;
    const auto k = nt ? zz_fp8_tiles_kernel<T, RO, RS, true> : zz_fp8_tiles_kernel<T, RO, RS, false>;
    hipLaunchKernelGGL(k, dim3((unsigned)g), dim3(C::NT), (C::LDS > P::LDS ? C::LDS : P::LDS), st, a, (int)whole);
    return true;
}

template <typename T, int RG, int RS, int NW, bool PF, bool NT>
static bool launch_few(const ZzF8Mm &a, hipStream_t st) {
    const dim3 g((a.m.O + 32 * RG - 1) / (32 * RG), (a.S + 32 * RS - 1) / (32 * RS));
    hipLaunchKernelGGL((zz_fp8_few_kernel<T, RG, RS, NW, PF, NT>), g, dim3(64 * NW), NW * RG * RS * 4096, st, a);
    return true;
}

// Which form: the one that is expected to take the shortest. A form's workgroups go round by
// round through the 256 CUs, `per` of them on a CU at once; a round with k workgroups on the
// busiest CU takes fix[k-1] + slope[k-1] * (blocks that a K group runs) microseconds. A form with
// `parts` runs what is over a multiple of 256 tiles in that many parts each, if these are at most
// one a CU: 2.9 + 0.49 * blocks after a full round, or less beside workgroups that are there
// (`busy`: fixed, a block, a block with a part on each CU). Fitted to 114 shapes (O 704 to 65536,
// I 256 to 8192, S 1 to 8192) with an rms error of 6 to 17 %. Over them the choice lies 2 % behind
// the best form of each, and up to 17 %. Any one form for all loses far more: the first and the
// last but one take 4.8 and 25.6 us for 1 x 4224 x 2816, 295 and 109 for 4096 rows; without the
// parts 4096 x 4224 x 2816 takes 107 us where it takes 95, 1000 x 4224 x 2816 36 for 30.
// The model has no bandwidth in it and holds for what it was fitted to. For few rows of matrices
// past the caches its times lie below what their bytes take (262144 x 4096: 131 us, where a read at
// 7.1 TB/s takes 151), and from about 3700 columns on it prefers the third form, whose loads go
// through the caches: 1 row of 262144 x 4096 180 us (6.0 TB/s), of 128256 x 7168 152 (6.1), of 18432
// x 7168 30 (4.4), where the second form's past the caches reaches 6.9 at 262144 x 2816.
struct ZzF8Form { int o, s, ks, per; float fix[4], slope[4]; int parts; float busy[3]; };
static const ZzF8Form mm_forms[] = {
    {32, 32, 16, 1, {1.9f}, {2.0f}},
    {32, 32, 4, 4, {2.9f, 2.3f, 2.6f, 0.7f}, {0.52f, 1.14f, 1.64f, 2.11f}},
    {64, 32, 8, 1, {2.6f}, {1.4f}},
    {64, 32, 2, 4, {2.8f, 3.2f, 2.9f, 2.5f}, {0.64f, 0.80f, 1.16f, 1.43f}},
    {64, 64, 4, 1, {3.4f}, {1.14f}},
    {64, 64, 2, 2, {3.0f, 2.8f}, {0.82f, 1.14f}},
    {64, 64, 1, 3, {2.8f, 3.9f, 2.1f}, {0.49f, 0.66f, 0.95f}},
    {64, 128, 1, 3, {3.4f, 6.0f, 4.0f}, {0.74f, 0.96f, 1.49f}},
    {64, 128, 1, 3, {3.4f, 6.0f, 4.0f}, {0.74f, 0.96f, 1.49f}, 2, {0.2f, 0.05f, 0.10f}},
    {128, 128, 1, 2, {4.5f, 7.8f}, {1.04f, 1.59f}},
    {128, 128, 1, 2, {4.5f, 7.8f}, {1.04f, 1.59f}, 4, {1.6f, 0.03f, 0.13f}},
    // zz_fp8_wide.h's, from 512 and 2816 columns with one to `per` workgroups on each CU
    {64, 64, 1, 4, {4.6f, 5.6f, 6.5f, 6.9f}, {0.41f, 0.45f, 0.48f, 0.62f}},
    {128, 64, 1, 3, {5.1f, 6.6f, 7.6f}, {0.46f, 0.58f, 0.81f}},
    {128, 128, 1, 2, {7.8f, 9.2f}, {0.63f, 0.93f}},
};
int zz_fp8_form(int O, int S, int tables, int nb, int of) {
    int best = 0;
    float least = INFINITY;
    // up to 32 rows the first three: the others' tiles are half empty
    for (int v = 0; v < (S <= 32 ? 3 : of == ZZ_F8_FORMS_8BIT ? 14 : 11); v++) {
        const ZzF8Form &f = mm_forms[v];
        if ((of == ZZ_F8_FORMS_8BIT && v >= 6 && v < 11) || (of && f.parts)) continue;
        int64_t n = (int64_t)((O + f.o - 1) / f.o) * ((S + f.s - 1) / f.s) * tables;
        const int r = (nb + f.ks - 1) / f.ks, cap = 256 * f.per;
        float t = 0.0f;
        if (f.parts) {
            const int parts = (int)(n % 256) * f.parts;
            if (!parts || parts > 256) continue;
            n -= n % 256;
            t = n % cap ? f.busy[0] + (f.busy[1] + f.busy[2] * parts / 256.0f) * r : 2.9f + 0.49f * r;
        }
        const int rem = (int)(n % cap);
        t += (float)(n / cap) * (f.fix[f.per - 1] + f.slope[f.per - 1] * r);
        if (rem) t += f.fix[(rem - 1) / 256] + f.slope[(rem - 1) / 256] * r;
        if (t < least) {
            least = t;
            best = v;
        }
    }
    return best;
}

template <typename T>
static bool launch_mm(const ZzF8Mm &a, hipStream_t st) {
    const int v = zz_fp8_form(a.m.O, a.S, 1, a.nb, ZZ_F8_FORMS_PLAIN);
    if (v == 0) return launch_few<T, 1, 1, 16, false, false>(a, st);
    // a large matrix, read once, past the caches; the activation rows come from the L2 for each
    // workgroup again, which 64 matrix rows a workgroup halve (200000 x 2816: 4 rows 85 us and 89
    // with 64, 16 rows 104 and 93, 32 rows 130 and 108)
    if (v == 1 && a.S <= 32 && (int64_t)a.m.O * a.m.I >= ZZ_NT_BYTES)
        return a.S <= 8 ? launch_few<T, 1, 1, 8, true, true>(a, st) : launch_few<T, 2, 1, 4, true, true>(a, st);
    if (v == 1) return launch_few<T, 1, 1, 4, true, false>(a, st);
    if (v == 2) return launch_few<T, 2, 1, 8, false, false>(a, st);
    if (v == 3) return launch_async<T, 1, 1, 2, 1, 2, 2>(a, st);
    if (v == 4) return launch_async<T, 1, 2, 2, 1, 4, 2>(a, st);
    if (v == 5) return launch_async<T, 1, 2, 2, 1, 2, 2>(a, st);
    if (v == 6) return launch_async<T, 1, 1, 2, 2, 1, 3>(a, st);
    if (v <= 8) return launch_tiles<T, 1, 2>(a, v == 8, st);
    return launch_tiles<T, 2, 2>(a, v == 10, st);
}

int zz_launch_fp8_matmul(const ZzF8Mat &m, const uint8_t *q, const float *s, int S, int dtype, void *y,
                         int64_t ldy, hipStream_t st) {
    const ZzF8Mm a{m, q, s, S, zz_f8_nb(m.I), y, ldy};
    return (dtype == 0 ? launch_mm<float>(a, st) : launch_mm<zz_bf16>(a, st)) && hipGetLastError() == hipSuccess;
}
