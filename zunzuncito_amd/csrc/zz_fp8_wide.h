// zz_fp8_wide.h -- tiles of the fp8 product with an epilogue whose results are bf16: the codes go
// into v_mfma_f32_32x32x64_f8f6f4 as they are.
//
// That instruction adds products up in f32, but first cuts the eight of each 8 columns to 13 bits
// behind the leading one of their largest, towards zero (measured: beside 2^14, 3.5 counts as 2 in
// the same eight and as itself in another). A product has 8 bits, so that it loses something only
// below 2^-5 of the largest, and less than 2^-13 of it: 7 x 2^-13 = 8.5e-4 of the terms' magnitudes
// at worst, 1.4e-5 of the 2-norm over normally distributed codes and 5e-5 over all codes alike. A
// result's own rounding to bf16 is 1.7e-3 in the 2-norm and up to 2^-8, so that it hides this; f32
// results, which would show it, and few rows, whose time is the matrix's bytes, keep
// zz_fp8_mma.h's f16 products.
//
// Without the conversions and at twice the rate: 8192 x 2816 x 2112 64 us (1.52 PFLOP/s) where the
// f16 tiles take 115; 2048 x 4224 x 2816 gated 39.5 for 71; 32768 rows of 128 experts, 1408 x 2816,
// 160 for 263. What bounds them is the way of the codes into LDS: the last without it takes 126 us,
// without the matrix instructions 157 (their clock is 1.9 GHz then; busy 39 %). Measured and not
// better, 128 x 128 tiles at 160: 256 x 256, one workgroup a CU (166; 12 % faster where the tiles
// come out even, 20 % slower where not), 64 x 64 a wave (170), operands of the next block read
// ahead over the barrier (170), later lines touched for the L2 (199 and more).
#pragma once
#include "zz_fp8_mma.h"

typedef int zz_i8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ zz_i8 zz_f8_pair(const char *a, const char *b) {
    const zz_u4 u = *(const zz_u4 *)a, v = *(const zz_u4 *)b;
    return zz_i8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
}

// 8 results as bf16 (v_cvt_pk_bf16_f32: to nearest even, a NaN stays one), n of them inside the
// row; nt: past the caches
__device__ __forceinline__ void zz_f8_store_bf16(zz_bf16 *p, const float (&v)[8], int n, bool nt) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    typedef float two __attribute__((ext_vector_type(2)));
    zz_u4 w;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = __builtin_bit_cast(unsigned, __builtin_convertvector(two{v[2 * j], v[2 * j + 1]}, pair));
    if (n >= 8) {
        if (nt) __builtin_nontemporal_store((zz_u4any)w, (zz_u4any *)p);
        else *(zz_u4any *)p = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 7; e++)
        if (e < n) p[e].u = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
}

// WO x WS waves of RO groups of 32 packed rows times 32 rows each
template <int RO, int WO, int WS>
struct ZzF8Wide {
    static constexpr int GW = WO * WS, NT = 64 * GW, O = 32 * RO * WO, S = 32 * WS;
    static constexpr int WB = O * 128, XB = S * 128, SI = (S + 63) / 64, STAGE = WB + XB + SI * 256;
    static constexpr int LDS = 2 * STAGE > O * S * 4 ? 2 * STAGE : O * S * 4;    // two blocks, or the result
    static constexpr int WI = O / 8 / GW, XI = S / 8 / GW;                       // a wave's requests a block
    static_assert(O / 8 % GW == 0 && S / 8 % GW == 0 && SI <= GW, "whole requests a wave");
};

// One tile: the result's rows from t0, the matrix's groups from gt. Blocks arrive in LDS as in
// zz_fp8_tile, one round ahead. A product's 16 results enter the sums while the next one runs, the
// last one's of a block behind the next barrier (with one group a wave, its own).
template <int G, int RO, int WO, int WS>
__device__ __forceinline__ void zz_fp8_wide(const ZzF8Ep &a, char *lds, int gt, int t0) {
    constexpr int GC = zz_f8_gw<G>;
    typedef ZzF8Wide<RO, WO, WS> C;
    const int tid = threadIdx.x, l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int w = zz_wave_id(), wo = w % WO, ws = w / WO;
    const int g0 = gt + wo * RO, gl = (a.m.O + GC - 1) / GC - 1, last = a.S - 1 - t0;
    const float *wsp = a.m.ws + (size_t)(min(g0, gl) / (128 / GC)) * nb, *wup = wsp;
    if constexpr (G == 2) wup += a.wsu;
    const unsigned lb = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    // this wave's requests: matrix pieces w*WI .. (4 a group), row octets w*XI .., the first waves'
    // 64 scales
    const uint8_t *wsrc[C::WI];
#pragma unroll
    for (int i = 0; i < C::WI; i++) {
        const int pc = w * C::WI + i;
        wsrc[i] = a.m.w + (size_t)min(gt + pc / 4, gl) * nb * 4096 + pc % 4 * 1024;
    }
    // (rows by index lie within 2^32 bytes of the first)
    const bool by_row = a.row != nullptr;
    const uint8_t *xsrc = a.q + (by_row ? 0 : (size_t)t0 * nb * ZZ_F8B);
    const float *ssrc = a.s + (by_row ? 0 : t0);
    ZzF8Scales wsl(wsp, nb), wul(wup, nb);
    unsigned xo[C::XI + 1];
#pragma unroll
    for (int i = 0; i < C::XI; i++) xo[i] = min((w * C::XI + i) * 8 + (l >> 3), last);
    xo[C::XI] = min(w * 64 + l, last);
    zz_f8_rows<G>(a, t0, xo);
    const unsigned so = 4 * xo[C::XI];
#pragma unroll
    for (int i = 0; i < C::XI; i++)
        xo[i] = xo[i] * nb * ZZ_F8B + 16 * ((l & 7) ^ ((((w * C::XI + i) & 1) << 2) | (l >> 4)));
    auto fetch = [&](int b) {
        const unsigned d = lb + (b & 1) * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::WI; i++) zz_dma16(wsrc[i] + (size_t)b * 4096, l * 16, d + (w * C::WI + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::XI; i++) zz_dma16(xsrc + (size_t)b * ZZ_F8B, xo[i], d + C::WB + (w * C::XI + i) * 1024);
        if (w < C::SI) zz_dma4(ssrc + (size_t)b * a.R, so, d + C::WB + C::XB + w * 256);
    };
    zz_v16f acc[RO], p[RO];
#pragma unroll
    for (int i = 0; i < RO; i++) acc[i] = p[i] = zz_f8_zero();
    float late = 0.0f, late2 = 0.0f;
    auto add = [&](int i, float sc, float sc2) {
#pragma unroll
        for (int k = 0; k < 16; k++) acc[i][k] = fmaf(p[i][k], k < 8 ? sc : sc2, acc[i][k]);
    };
    fetch(0);
    wsl.ready();
    wul.ready();
    for (int b = 0; b < nb; b++) {
        // block b has arrived for this wave; behind the barrier, for all, and the one before it is read
        zz_wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (b + 1 < nb) fetch(b + 1);
        const char *d = lds + (b & 1) * C::STAGE;
        const int t = ws * 32 + r;
        zz_i8 wv[RO][2], xv[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const char *q = d + C::WB + t * 128;
            xv[k] = zz_f8_pair(q + 16 * ((4 * k + h) ^ ((r >> 1) & 7)), q + 16 * ((4 * k + 2 + h) ^ ((r >> 1) & 7)));
#pragma unroll
            for (int i = 0; i < RO; i++) {
                const char *c = d + ((wo * RO + i) * 4 + 2 * k) * 1024 + l * 16;
                wv[i][k] = zz_f8_pair(c, c + 1024);
            }
        }
        const float xsc = *(const float *)(d + C::WB + C::XB + 4 * t);
        const float sc = xsc * wsl.of(b), sc2 = G == 2 ? xsc * wul.of(b) : sc;
#pragma unroll
        for (int i = 0; i < RO; i++) {
            __builtin_amdgcn_sched_barrier(0);
            p[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[i][0], xv[0], zz_f8_zero(), 0, 0, 0, 0, 0, 0);
            p[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[i][1], xv[1], p[i], 0, 0, 0, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (RO == 1) add(0, sc, sc2);
            else if (i) add(i - 1, sc, sc2);
            else add(RO - 1, late, late2);
        }
        late = sc;
        late2 = sc2;
    }
    if constexpr (RO > 1) add(RO - 1, late, late2);
    // The tile goes through LDS, [row][packed row] in 16-byte pieces (a row's pieces permuted by the
    // row, for the banks), and leaves in whole lines.
    float *tile = (float *)lds;
    auto place = [&](int t, int o) { return tile + t * C::O + 4 * ((((o >> 2) ^ t) & 7) | ((o >> 2) & ~7)); };
    __syncthreads();                                      // the last block is read
#pragma unroll
    for (int i = 0; i < RO; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
            *(float4 *)place(ws * 32 + r, (wo * RO + i) * 32 + 8 * k + 4 * h) =
                make_float4(acc[i][4 * k], acc[i][4 * k + 1], acc[i][4 * k + 2], acc[i][4 * k + 3]);
    __syncthreads();
    constexpr int RL = C::O / 32 * GC / 8;                // lanes a row
    for (int q = tid; q < C::S * RL; q += C::NT) {
        const int t = q / RL, o = q % RL * 8, from = o / GC * 32 + o % GC, col = GC * gt + o, n = a.m.O - col;
        if (t > last) break;
        if (n <= 0) continue;
        float v[8], u[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *(float4 *)(v + e) = *(const float4 *)place(t, from + e);
            if constexpr (G == 2) *(float4 *)(u + e) = *(const float4 *)place(t, from + 16 + e);
        }
        zz_f8_end<G>(a, v, u, col, n, (const zz_bf16 *)a.res + (int64_t)(t0 + t) * a.ldr + col);
        zz_f8_store_bf16((zz_bf16 *)a.y + (int64_t)(t0 + t) * a.ldy + col, v, n, a.nt);
    }
}

// OCC: waves a SIMD, so that three or four tiles, two of the largest, share a CU
template <int G, int RO, int WO, int WS, int OCC>
__global__ __launch_bounds__(64 * WO * WS, OCC) void zz_fp8_wide_kernel(ZzF8Ep a) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    typedef ZzF8Wide<RO, WO, WS> C;
    int ot, st;
    if (!zz_f8_place<G, zz_bf16, C::O / 32, C::S>(a, &ot, &st)) return;
    zz_fp8_wide<G, RO, WO, WS>(a, lds, ot * C::O / 32, st * C::S);
}

template <int G, int RO, int WO, int WS, int OCC>
static bool launch_wide(const ZzF8EpCall &c, const ZzF8Ep &a, hipStream_t st) {
    return launch_tiles_ep<ZzF8Wide<RO, WO, WS>, G>(c, a, zz_fp8_wide_kernel<G, RO, WO, WS, OCC>, st);
}
