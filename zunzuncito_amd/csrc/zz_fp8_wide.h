// zz_fp8_wide.h -- tiles of the fp8 product with an epilogue whose results are bf16, where the
// caller takes sums of fewer bits (ZZ_EP_8BIT): the codes go into v_mfma_f32_32x32x64_f8f6f4 as
// they are.
//
// That instruction adds products up in f32, but first cuts the eight of each 8 columns to 13 bits
// behind the leading one of their largest, towards zero (measured: beside 2^14, 3.5 counts as 2 in
// the same eight and as itself in another). A product has 8 bits, so that it loses something only
// below 2^-5 of the largest, and less than 2^-13 of it: 7 x 2^-13 = 8.5e-4 of the terms' magnitudes
// at worst, 1.4e-5 of the 2-norm over normally distributed codes and 5e-5 over all codes alike. A
// result's own rounding to bf16 is 1.7e-3 in the 2-norm and up to 2^-8, which hides this unless
// the terms cancel: then nothing may be left (2^14 - 2^14 + 36, the 36 from four products beside
// the first, comes out as 0). So no call has these tiles that does not ask for them; f32
// results, which would show the cut, and few rows, whose time is the matrix's bytes, keep
// zz_fp8_mma.h's f16 products all the same.
//
// Without the conversions and at twice the rate: 8192 x 2816 x 2112 65 us (1.50 PFLOP/s) where the
// f16 tiles take 115; 2048 x 4224 x 2816 gated 36.8 for 66; 32768 rows of 128 experts, 1408 x 2816, 256
// each 204 for 298, all of 8 experts 161 for 295. Nothing is full (in the order of the last three): the
// matrix cores are 25, 31 and 40 % busy, LDS's index path 16, 20 and 26 % with conflicts below 1 %, of
// memory 1.4 TB/s are asked. Two waves a SIMD wait for each other's round, and at a tile's start and end.
// A wave keeps 32 packed rows times all rows of the tile: its part of the matrix lies in operand order, no
// other wave wants it, and it comes straight into registers, past LDS, which then holds more blocks. With the matrix
// through LDS and waves of 64 x 32 128 experts of 256 rows each took 224 for 197, 64 of 512 188 for 169, 64
// rows each 125 for 120. Measured and not better (8 experts of 4096 rows, 128 x 128 at 164): 256 x 256 (166)
// and 256 x 128 (184), 64 x 64 a wave (170), a third workgroup on a
// CU (spills), the row operands' next block read over the barrier (170), later lines touched for the
// L2 (199 and more), the XCDs' parts cut by the matrices they read (171: more workgroups without a tile).
#pragma once
#include "zz_fp8_mma.h"
#include <type_traits>

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

// WO waves of 32 packed rows times 32 RS rows each
template <int RS, int WO>
struct ZzF8Wide {
    static constexpr int NT = 64 * WO, O = 32 * WO, S = 32 * RS;
    static constexpr int XB = S * 128, SI = (S + 63) / 64, STAGE = XB + SI * 256;
    static constexpr int LDS = 2 * STAGE > O * S * 4 ? 2 * STAGE : O * S * 4;    // two blocks, or the result
    static constexpr int XI = S / 8 / WO;                                        // a wave's requests a block
    static_assert(S / 8 % WO == 0 && SI <= WO, "whole requests a wave");
};

// One tile: the result's rows from t0, the matrix's groups from gt. The rows' blocks arrive in LDS
// as in zz_fp8_tile, one round ahead; the matrix's in registers, two rounds ahead. A product's 16
// results enter the sums while the next one runs, the last one's of a block behind the next barrier.
template <int G, int RS, int WO>
__device__ __forceinline__ void zz_fp8_wide(const ZzF8Ep &a, char *lds, int gt, int t0) {
    constexpr int GC = zz_f8_gw<G>;
    typedef ZzF8Wide<RS, WO> C;
    const int tid = threadIdx.x, l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb, w = zz_wave_id();
    const int gl = (a.m.O + GC - 1) / GC - 1, g0 = min(gt + w, gl), last = a.S - 1 - t0;
    const float *wsp = a.m.ws + (size_t)(g0 / (128 / GC)) * nb, *wup = wsp;
    if constexpr (G == 2) wup += a.wsu;
    const unsigned lb = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const uint8_t *wsrc = a.m.w + (size_t)g0 * nb * 4096;
    // this wave's requests: row octets w*XI .., the first waves' 64 scales
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
        for (int i = 0; i < C::XI; i++) zz_dma16(xsrc + (size_t)b * ZZ_F8B, xo[i], d + (w * C::XI + i) * 1024);
        if (w < C::SI) zz_dma4(ssrc + (size_t)b * a.R, so, d + C::XB + w * 256);
    };
    struct Codes { zz_u4 v[4]; } w0, w1, w2;
    auto ask = [&](Codes &c, int b) {                     // behind the last block: its data, not used
        const uint8_t *from = wsrc + (size_t)min(b, nb - 1) * 4096 + l * 16;
#pragma unroll
        for (int k = 0; k < 4; k++) c.v[k] = *(const zz_u4 *)(from + k * 1024);
    };
    zz_v16f acc[RS], p[2] = {zz_f8_zero(), zz_f8_zero()};
#pragma unroll
    for (int j = 0; j < RS; j++) acc[j] = zz_f8_zero();
    float late = 0.0f, late2 = 0.0f;
    auto add = [&](int j, float sc, float sc2) {
#pragma unroll
        for (int k = 0; k < 16; k++) acc[j][k] = fmaf(p[j & 1][k], k < 8 ? sc : sc2, acc[j][k]);
        asm volatile("" : "+v"(acc[j]));                  // here, not where the sums are read next
    };
    // A round requests the next block's rows, then the codes of the matrix for the one after it:
    // before block b what may be on its way are the four requests for the codes of block b + 1, the
    // youngest. LEFT is their number, 0 behind which nothing was requested.
    auto round = [&](int b, Codes &wc, auto LEFT, auto next) {
        // block b has arrived for this wave; behind the barrier, for all, and the one before it is read
        zz_wait_vm<LEFT.value>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        zz_i8 wv[2];
#pragma unroll
        for (int k = 0; k < 4; k++) asm volatile("" : "+v"(wc.v[k]));
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const zz_u4 u = wc.v[2 * k], v = wc.v[2 * k + 1];
            wv[k] = zz_i8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (b + 1 < nb) fetch(b + 1);
        asm volatile("" ::: "memory");
        next(b + 2);
        asm volatile("" ::: "memory");
        const char *d = lds + (b & 1) * C::STAGE;
        zz_i8 xv[2][2];
        auto operand = [&](int j) {
            const char *q = d + (j * 32 + r) * 128;
#pragma unroll
            for (int k = 0; k < 2; k++)
                xv[j & 1][k] = zz_f8_pair(q + 16 * ((4 * k + h) ^ ((r >> 1) & 7)), q + 16 * ((4 * k + 2 + h) ^ ((r >> 1) & 7)));
        };
        operand(0);
        float sc[RS], sc2[RS];
        const float wsc = wsl.of(b), wsc2 = G == 2 ? wul.of(b) : wsc;
#pragma unroll
        for (int j = 0; j < RS; j++) {
            const float xsc = *(const float *)(d + C::XB + 4 * (j * 32 + r));
            sc[j] = xsc * wsc;
            sc2[j] = G == 2 ? xsc * wsc2 : sc[j];
        }
#pragma unroll
        for (int j = 0; j < RS; j++) {
            if (j + 1 < RS) operand(j + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; k++)
                p[j & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[k], xv[j & 1][k], k ? p[j & 1] : zz_f8_zero(), 0, 0, 0, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (j) add(j - 1, sc[j - 1], sc2[j - 1]);
            else add(RS - 1, late, late2);
        }
        late = sc[RS - 1];
        late2 = sc2[RS - 1];
    };
    std::integral_constant<int, 4> four;
    std::integral_constant<int, 0> none;
    ask(w0, 0);
    asm volatile("" ::: "memory");
    fetch(0);
    asm volatile("" ::: "memory");
    ask(w1, 1);
    asm volatile("" ::: "memory");
    wsl.ready();
    wul.ready();
    // in threes, so that no register is moved before it is there; a round skipped inside the loop
    // would have the compiler wait for the youngest codes
    int b = 0;
    for (; b + 3 <= nb; b += 3) {
        round(b, w0, four, [&](int n) { ask(w2, n); });
        round(b + 1, w1, four, [&](int n) { ask(w0, n); });
        round(b + 2, w2, four, [&](int n) { ask(w1, n); });
    }
    if (b < nb) round(b, w0, four, [](int) {});
    if (b + 1 < nb) round(b + 1, w1, none, [](int) {});
    add(RS - 1, late, late2);
    // The tile goes through LDS, [row][packed row] in 16-byte pieces (a row's pieces permuted by the
    // row, for the banks), and leaves in whole lines.
    float *tile = (float *)lds;
    auto place = [&](int t, int o) { return tile + t * C::O + 4 * ((((o >> 2) ^ t) & 7) | ((o >> 2) & ~7)); };
    __syncthreads();                                      // the last block is read
#pragma unroll
    for (int j = 0; j < RS; j++)
#pragma unroll
        for (int k = 0; k < 4; k++)
            *(float4 *)place(j * 32 + r, w * 32 + 8 * k + 4 * h) =
                make_float4(acc[j][4 * k], acc[j][4 * k + 1], acc[j][4 * k + 2], acc[j][4 * k + 3]);
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

// OCC: waves a SIMD that the registers are to allow
template <int G, int RS, int WO, int OCC>
__global__ __launch_bounds__(64 * WO, OCC) void zz_fp8_wide_kernel(ZzF8Ep a) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    typedef ZzF8Wide<RS, WO> C;
    int ot, st;
    if (!zz_f8_place<G, zz_bf16, C::O / 32, C::S>(a, &ot, &st)) return;
    zz_fp8_wide<G, RS, WO>(a, lds, ot * C::O / 32, st * C::S);
}

template <int G, int RS, int WO, int OCC>
static bool launch_wide(const ZzF8EpCall &c, const ZzF8Ep &a, hipStream_t st) {
    return launch_tiles_ep<ZzF8Wide<RS, WO>, G>(c, a, zz_fp8_wide_kernel<G, RS, WO, OCC>, st);
}
