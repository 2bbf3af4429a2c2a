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
// there are fewer than pieces. Pieces can be more than a launch's threads.
__global__ __launch_bounds__(256) void zz_fp8_pack_kernel(const uint8_t *src, int O, int I, int nb, uint8_t *dst,
                                                          int64_t n, int part, const float *scales, float *ws, int ns) {
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < n; p += (int64_t)gridDim.x * 256) {
        if (p < ns) ws[p] = scales[p];
        const int l = (int)(p & 63), pc = (int)(p >> 6) & 3;
        const int64_t gb = p >> 8, g = gb / nb;
        const int b = (int)(gb - g * nb), k = b * ZZ_F8B + 32 * pc + 16 * (l >> 5);
        int64_t row = g * 32 + (l & 31);
        if (part >= 0) {
            if (((l >> 4) & 1) != part) continue;
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
}

int zz_launch_fp8_pack(const uint8_t *codes, int O, int I, int part, uint8_t *dst, const float *scales, float *ws, hipStream_t st) {
    const int nb = zz_f8_nb(I), gc = part < 0 ? 32 : 16;
    const int64_t n = (int64_t)((O + gc - 1) / gc) * nb * 256;
    const int64_t g = (n + 255) / 256, most = 1 << 23;    // 2^31 threads
    hipLaunchKernelGGL(zz_fp8_pack_kernel, dim3((unsigned)(g < most ? g : most)), dim3(256), 0, st, codes, O, I, nb, dst, n, part,
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
