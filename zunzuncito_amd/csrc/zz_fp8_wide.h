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
// Without the conversions and at twice the rate: 8192 x 2816 x 2112 62.7 us (1.55 PFLOP/s) where the
// f16 tiles take 115; 2048 x 4224 x 2816 gated 40 for 71; 32768 rows of 128 experts, 1408 x 2816,
// 176 for 263.
#pragma once
#include "zz_fp8_mma.h"

typedef int zz_i8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ zz_i8 zz_f8_pair(zz_u4 a, zz_u4 b) {
    return zz_i8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
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

template <int RO, int RS, int WO, int WS, int NS>
struct ZzF8Wide {
    static constexpr int GW = WO * WS, NT = 64 * GW, O = 32 * RO * WO, S = 32 * RS * WS;
    static constexpr int WB = O * 128, XB = S * 128, SB = S * 4 < 256 ? 256 : S * 4, STAGE = WB + XB + SB;
    static constexpr int PART = 32 * WS * O * 4;          // bytes of the part of the result that leaves at once
    static constexpr int LDS = NS * STAGE > (RS > 1 ? 2 : 1) * PART ? NS * STAGE : (RS > 1 ? 2 : 1) * PART;
    static constexpr int WI = O / 8 / GW, XI = S / 8 / GW, DMA = WI + XI + 1;   // a wave's requests a block
    static_assert(O / 8 % GW == 0 && S / 8 % GW == 0 && SB / 256 <= GW, "whole requests a wave");
};

// One tile: the result's rows from t0, the matrix's groups from gt. Blocks arrive in LDS as in
// zz_fp8_tile. A wave keeps its RO groups' codes of a block and goes through its RS row tiles; a
// product's 16 results enter the sums while the next one runs, the last of a block's behind the
// barrier.
template <int G, int RO, int RS, int WO, int WS, int NS>
__device__ __forceinline__ void zz_fp8_wide(const ZzF8Ep &a, char *lds, int gt, int t0) {
    constexpr int GC = zz_f8_gw<G>;
    typedef ZzF8Wide<RO, RS, WO, WS, NS> C;
    const int tid = threadIdx.x, l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int w = zz_wave_id(), wo = w % WO, ws = w / WO;
    const int g0 = gt + wo * RO, gl = (a.m.O + GC - 1) / GC - 1, last = a.S - 1 - t0;
    const float *wsp = a.m.ws + (size_t)(min(g0, gl) / (128 / GC)) * nb, *wup = wsp;
    if constexpr (G == 2) wup += a.wsu;
    const unsigned lb = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const uint8_t *wsrc[C::WI];
#pragma unroll
    for (int i = 0; i < C::WI; i++) {
        const int pc = w * C::WI + i;
        wsrc[i] = a.m.w + (size_t)min(gt + pc / 4, gl) * nb * 4096 + pc % 4 * 1024;
    }
    const bool by_row = a.row != nullptr;
    const uint8_t *xsrc = a.q + (by_row ? 0 : (size_t)t0 * nb * ZZ_F8B);
    const float *ssrc = a.s + (by_row ? 0 : t0);
    auto at = [&](int t) {
        const int in = min(t, last);
        return (unsigned)(by_row ? zz_f8_row<G>(a, t0 + in) : in);
    };
    unsigned xo[C::XI];
#pragma unroll
    for (int i = 0; i < C::XI; i++)
        xo[i] = at((w * C::XI + i) * 8 + (l >> 3)) * nb * ZZ_F8B + 16 * ((l & 7) ^ ((((w * C::XI + i) & 1) << 2) | (l >> 4)));
    constexpr int SI = C::SB / 256;
    const unsigned so = 4 * at(w % SI * 64 + l);
    auto fetch = [&](int b, int slot) {
        const unsigned d = lb + slot * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::WI; i++) zz_dma16(wsrc[i] + (size_t)b * 4096, l * 16, d + (w * C::WI + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::XI; i++) zz_dma16(xsrc + (size_t)b * ZZ_F8B, xo[i], d + C::WB + (w * C::XI + i) * 1024);
        zz_dma4(ssrc + (size_t)b * a.R, so, d + C::WB + C::XB + w % SI * 256);
    };
    ZzF8Scales wsl(wsp, nb), wul(wup, nb);
    zz_v16f acc[RO][RS];
#pragma unroll
    for (int i = 0; i < RO; i++)
#pragma unroll
        for (int j = 0; j < RS; j++) acc[i][j] = zz_f8_zero();
#pragma unroll
    for (int i = 0; i < NS - 1; i++)
        if (i < nb) fetch(i, i);
    zz_v16f p[RO];
    p[RO - 1] = zz_f8_zero();
    float late = 0.0f, late2 = 0.0f;
    int slot = 0, into = NS - 1;
    for (int b = 0; b < nb; b++) {
        if (b + NS - 2 < nb) zz_wait_vm<C::DMA *(NS - 2)>();
        else zz_wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (b + NS - 1 < nb) fetch(b + NS - 1, into);
        const char *d = lds + slot * C::STAGE;
        slot = slot + 1 == NS ? 0 : slot + 1;
        into = into + 1 == NS ? 0 : into + 1;
        const float wsc = wsl.of(b), wsc2 = G == 2 ? wul.of(b) : wsc;
        zz_i8 wv[RO][2], xn[2];
        float sn;
        auto rows = [&](int j) {                          // row tile j's codes and scale
            const int t = (ws * RS + j) * 32 + r;
            const char *q = d + C::WB + t * 128;
#pragma unroll
            for (int k = 0; k < 2; k++)
                xn[k] = zz_f8_pair(*(const zz_u4 *)(q + 16 * ((4 * k + h) ^ ((r >> 1) & 7))),
                                   *(const zz_u4 *)(q + 16 * ((4 * k + 2 + h) ^ ((r >> 1) & 7))));
            sn = *(const float *)(d + C::WB + C::XB + 4 * t);
        };
#pragma unroll
        for (int i = 0; i < RO; i++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const char *q = d + ((wo * RO + i) * 4 + 2 * k) * 1024 + l * 16;
                wv[i][k] = zz_f8_pair(*(const zz_u4 *)q, *(const zz_u4 *)(q + 1024));
            }
        rows(0);
#pragma unroll
        for (int j = 0; j < RS; j++) {
            const zz_i8 xv[2] = {xn[0], xn[1]};
            const float sc = sn * wsc, sc2 = G == 2 ? sn * wsc2 : sc;
            if (j + 1 < RS) rows(j + 1);
#pragma unroll
            for (int i = 0; i < RO; i++) {
                __builtin_amdgcn_sched_barrier(0);
                p[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[i][0], xv[0], zz_f8_zero(), 0, 0, 0, 0, 0, 0);
                p[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[i][1], xv[1], p[i], 0, 0, 0, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                // the product before this one enters its sums meanwhile (with one group, this one)
                const int pi = i ? i - 1 : RO - 1, pj = i || RO == 1 ? j : j ? j - 1 : RS - 1;
                const float ps = i || RO == 1 ? sc : late, ps2 = i || RO == 1 ? sc2 : late2;
#pragma unroll
                for (int k = 0; k < 16; k++) acc[pi][pj][k] = fmaf(p[pi][k], k < 8 ? ps : ps2, acc[pi][pj][k]);
            }
            __builtin_amdgcn_sched_barrier(0);
            late = sc;
            late2 = sc2;
        }
    }
    if constexpr (RO > 1)
#pragma unroll
        for (int k = 0; k < 16; k++) acc[RO - 1][RS - 1][k] = fmaf(p[RO - 1][k], k < 8 ? late : late2, acc[RO - 1][RS - 1][k]);
    // 32 WS rows at a time go through LDS, [row][packed row] in 16-byte pieces (a row's pieces
    // permuted by the row, for the banks), and leave in whole lines.
    constexpr int CO = C::O / 32 * GC, RL = CO / 8;       // columns, lanes a row
#pragma unroll 1
    for (int j = 0; j < RS; j++) {
        float *tile = (float *)(lds + (j & 1) * C::PART);
        auto place = [&](int t, int o) { return tile + t * C::O + 4 * ((((o >> 2) ^ t) & 7) | ((o >> 2) & ~7)); };
        if (j == 0) __syncthreads();                      // the last block is read
#pragma unroll
        for (int f = 0; f < RS; f++)
            if (f == j)
#pragma unroll
                for (int i = 0; i < RO; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        *(float4 *)place(ws * 32 + r, (wo * RO + i) * 32 + 8 * k + 4 * h) =
                            make_float4(acc[i][f][4 * k], acc[i][f][4 * k + 1], acc[i][f][4 * k + 2], acc[i][f][4 * k + 3]);
        __syncthreads();                                  // (and the part before the last is read)
        for (int q = tid; q < 32 * WS * RL; q += C::NT) {
            const int in = q / RL, o = q % RL * 8, from = o / GC * 32 + o % GC, col = GC * gt + o, n = a.m.O - col;
            const int t = (in / 32 * RS + j) * 32 + in % 32;
            if (t > last || n <= 0) continue;
            float v[8], u[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                *(float4 *)(v + e) = *(const float4 *)place(in, from + e);
                if constexpr (G == 2) *(float4 *)(u + e) = *(const float4 *)place(in, from + 16 + e);
            }
            zz_f8_end<G>(a, v, u, col, n, (const zz_bf16 *)a.res + (int64_t)(t0 + t) * a.ldr + col);
            zz_f8_store_bf16((zz_bf16 *)a.y + (int64_t)(t0 + t) * a.ldy + col, v, n, a.nt);
        }
    }
}

template <int G, int RO, int RS, int WO, int WS, int NS, int OCC>
__global__ __launch_bounds__(64 * WO * WS, OCC) void zz_fp8_wide_kernel(ZzF8Ep a) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    typedef ZzF8Wide<RO, RS, WO, WS, NS> C;
    int ot, st;
    if (!zz_f8_place<G, zz_bf16, C::O / 32, C::S>(a, &ot, &st)) return;
    zz_fp8_wide<G, RO, RS, WO, WS, NS>(a, lds, ot * C::O / 32, st * C::S);
}

template <int G, int RO, int RS, int WO, int WS, int NS, int OCC>
static bool launch_wide(const ZzF8EpCall &c, const ZzF8Ep &a, hipStream_t st) {
    typedef ZzF8Wide<RO, RS, WO, WS, NS> C;
    return launch_tiles_ep<C, G>(c, a, zz_fp8_wide_kernel<G, RO, RS, WO, WS, NS, OCC>, st);
}
