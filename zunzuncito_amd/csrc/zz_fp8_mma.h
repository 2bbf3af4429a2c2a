// zz_fp8_mma.h -- the device code of the products of e4m3 rows with resident e4m3 matrices
// (include/zz_fp8.h): zz_fp8_mma.hip has one plain matrix, zz_fp8_ep.hip and zz_fp8_gated.hip
// what has an epilogue and tables of experts.
//
//   y[s][o] = sum_b xs[b][s] * ws[o/128][b] * sum_{k in block b} xq[s][k] wq[o][k]
// The codes are multiplied as f16, which holds every e4m3 value: the products are exact and
// the matrix core adds them up in f32. The 8-bit instructions do not (zz_fp8_wide.h): they are
// 1.4e-5 off in the 2-norm over normally distributed codes and up to 8.5e-4 of the terms' magnitudes,
// where the f16 form is 1e-8 and 2e-7 off, at twice the rate (8192^3 in a library 2.7 PFLOP/s, in
// f16 1.35). A product with an epilogue takes them where its caller allows it. bf16
// holds every code too, and its library product is faster (1.48): not tried.
//
// A block of 128 columns is eight v_mfma_f32_32x32x16_f16 of 32 matrix rows times 32
// activation rows; each of the 16 results a lane then enters the f32 accumulator by one fma
// with the two scales' product. Lane 32h + r holds activation row r and the matrix rows
// 8k + 4h .. + 3 (k = 0..3) of the group, so a lane needs one row scale and a group one matrix
// scale. (The 16x16x32 form leaves 3 of 4 issue slots to the conversions and fma's beside it,
// this one 7 of 8: with 3 vector operations for each 16 cycles of matrix work, as here, 24 and
// 19 cycles were measured.)
#pragma once
#include "zz_fp8_dev.h"
#include <math.h>
typedef _Float16 zz_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 zz_h8 __attribute__((ext_vector_type(8)));
typedef float zz_v16f __attribute__((ext_vector_type(16)));

// 8 codes (two words) as f16: v_cvt_scalef32_pk_f16_fp8 at scale 1, exact, NaN stays NaN
__device__ __forceinline__ zz_h8 zz_f8_half(unsigned a, unsigned b) {
    const zz_h2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, false);
    const zz_h2 q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, true);
    const zz_h2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, false);
    const zz_h2 t = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, true);
    return zz_h8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
}
// step e (0, 1) of a 16-byte piece
__device__ __forceinline__ zz_h8 zz_f8_step(uint4 v, int e) { return e ? zz_f8_half(v.z, v.w) : zz_f8_half(v.x, v.y); }

__device__ __forceinline__ zz_v16f zz_f8_zero() {
    zz_v16f z;
#pragma unroll
    for (int i = 0; i < 16; i++) z[i] = 0.0f;
    return z;
}

// matrix rows o..o+3 of activation row t
template <typename T>
__device__ __forceinline__ void zz_f8_store4(T *y, int64_t ldy, int t, int o, int O, const float (&v)[4]) {
    T *p = y + (int64_t)t * ldy + o;
    if (o + 4 <= O) {
        if constexpr (sizeof(T) == 4)
            *(zz_u4any *)p = zz_u4any{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        else
            *(zz_u2any *)p = zz_u2any{zz_bf16_bits(v[0]) | zz_bf16_bits(v[1]) << 16, zz_bf16_bits(v[2]) | zz_bf16_bits(v[3]) << 16};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (o + i < O) zz_put(p + i, v[i]);
}

// 16 bytes of a result row, n of its elements inside the row
template <bool NT, typename T>
__device__ __forceinline__ void zz_f8_store(T *p, const float (&v)[16 / sizeof(T)], int n) {
    constexpr int E = 16 / sizeof(T);
    if (n >= E) {
        zz_u4any w;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if constexpr (E == 4) w[j] = __float_as_uint(v[j]);
            else w[j] = zz_bf16_bits(v[2 * j]) | zz_bf16_bits(v[2 * j + 1]) << 16;
        if constexpr (NT) __builtin_nontemporal_store(w, (zz_u4any *)p);
        else *(zz_u4any *)p = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < E; i++)
        if (i < n) zz_put(p + i, v[i]);
}

struct ZzF8Mm {
    ZzF8Mat m;
    const uint8_t *q;
    const float *s;
    int S, nb;
    void *y;
    int64_t ldy;
};

// What a product with an epilogue, or over a table of experts, has besides (forms G = 1, and 2
// for gated pairs). Matrices of a gated pair lie in one: group g of 32 packed rows is gate's rows
// 16g .. + 15, then up's, so that a lane's results 0-7 and 8-15 are the same columns of both.
struct ZzF8Ep : ZzF8Mm {
    int R;                      // rows of q, the distance of s's blocks
    const int *row;             // the row of q for each row of y, or null
    const float *bias;          // [O], gated [2][O]
    const void *res;
    int64_t ldr;
    int act;                    // ZZ_EP_*
    float clamp;
    int nt;                     // large tiles' results are stored past the caches
    const int *offs;            // [E + 1], or null: one matrix for all rows
    int E, P;
    int64_t we;                 // bytes of an expert's codes
    int wse, wsu;               // floats of an expert's scales, of gate's before up's
};

// packed rows of a group that are columns of y
template <int G> constexpr int zz_f8_gw = G == 2 ? 16 : 32;
// the distance of the rows' scales
template <int G, typename A>
__device__ __forceinline__ int zz_f8_stride(const A &a) {
    if constexpr (G) return a.R;
    else return a.S;
}
// the row of q for row t: an index from the outside, which may be anything
template <int G, typename A>
__device__ __forceinline__ int zz_f8_row(const A &a, int t) {
    if constexpr (G) {
        if (!a.row) return t;
        const int i = a.row[t];
        return (unsigned)i < (unsigned)a.R ? i : 0;
    } else {
        return t;
    }
}

// The same for N rows t0 + t[k] of a tile, their indexes requested together (one after the other, a
// tile began two microseconds later: 32768 rows to 8 of 128 experts, 1408 x 2816 gated, took 172 us for 160);
// without an index t stays as it is, from the tile's first row.
template <int G, int N, typename A>
__device__ __forceinline__ void zz_f8_rows(const A &a, int t0, unsigned (&t)[N]) {
    if constexpr (G)
        if (a.row) {
#pragma unroll
            for (int k = 0; k < N; k++) t[k] = (unsigned)a.row[t0 + (int)t[k]];
#pragma unroll
            for (int k = 0; k < N; k++) t[k] = t[k] < (unsigned)a.R ? t[k] : 0;
        }
}

// N (4 or 8) elements at any address as f32, n of them inside
template <int N, typename T>
__device__ __forceinline__ void zz_f8_load(float (&v)[N], const T *p, int n) {
    if (n >= N) {
        if constexpr (N == 4 && sizeof(T) == 2) {
            const zz_u2any a = *(const zz_u2any *)p;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __uint_as_float(j & 1 ? a[j >> 1] & 0xffff0000u : a[j >> 1] << 16);
        } else {
#pragma unroll
            for (int q = 0; q < N * (int)sizeof(T) / 16; q++) {
                const zz_u4 a = *((const zz_u4any *)p + q);
#pragma unroll
                for (int j = 0; j < 16 / (int)sizeof(T); j++)
                    if constexpr (sizeof(T) == 4) v[4 * q + j] = __uint_as_float(a[j]);
                    else v[8 * q + j] = __uint_as_float(j & 1 ? a[j >> 1] & 0xffff0000u : a[j >> 1] << 16);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < n ? zz_f32_of(p[i]) : 0.0f;
}

// N sums (gated: and up's) of columns o .. o + n - 1 to results: bias, activation, gate, residual
// (res: the row's at column o). One hardware exponential and one reciprocal a result; sums that
// are NaN stay so.
template <int G, int N, typename T>
__device__ __forceinline__ void zz_f8_end(const ZzF8Ep &a, float (&v)[N], float (&u)[N], int o, int n, const T *res) {
    float t[N];
    if (a.bias) {
        zz_f8_load(t, a.bias + o, n);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += t[i];
        if constexpr (G == 2) {
            zz_f8_load(t, a.bias + a.m.O + o, n);
#pragma unroll
            for (int i = 0; i < N; i++) u[i] += t[i];
        }
    }
    if (a.res) zz_f8_load(t, res, n);
    if constexpr (G == 2)
        if (a.clamp > 0.0f)
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i] = v[i] > a.clamp ? a.clamp : v[i];
                u[i] = u[i] > a.clamp ? a.clamp : u[i] < -a.clamp ? -a.clamp : u[i];
            }
    if (a.act == 1) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = zz_gelu_tanh(v[i]);
    } else if (a.act == 2) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = zz_silu(v[i]);
    }
    if constexpr (G == 2)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= u[i];
    if (a.res)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += t[i];
}

// Few rows: a workgroup per RG groups of 32 matrix rows and RS tiles of 32 activation rows;
// its NW waves take every NW-th block, straight from memory into registers (PF: the next one's
// codes requested before the current one is multiplied), and meet in LDS, where the partial
// sums are added in the waves' order. Rows behind the last one are read as the last one, and
// not stored. NT: the matrix is read once and does not stay in the caches: 3 rows against
// 262144 x 2816 in 104 us, 7.1 TB/s, instead of 120.
// part: [NW][RG][RS][16][64] in LDS; groups from g0, rows from t0.
template <typename T, int G, int RG, int RS, int NW, bool PF, bool NT, typename A>
__device__ __forceinline__ void zz_fp8_few(const A &a, float *part, int g0, int t0) {
    constexpr int GC = zz_f8_gw<G>;
    const int tid = threadIdx.x, w = zz_wave_id(), l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int gl = (a.m.O + GC - 1) / GC - 1, rs = zz_f8_stride<G>(a);
    const uint8_t *wp[RG], *xp[RS];
    const float *ws = a.m.ws + (size_t)(g0 / (128 / GC)) * nb, *wu = ws, *sp[RS];
    if constexpr (G == 2) wu += a.wsu;
#pragma unroll
    for (int i = 0; i < RG; i++) wp[i] = a.m.w + (size_t)min(g0 + i, gl) * nb * 4096 + l * 16;
#pragma unroll
    for (int j = 0; j < RS; j++) {
        const int t = zz_f8_row<G>(a, min(t0 + 32 * j + r, a.S - 1));
        xp[j] = a.q + (size_t)t * nb * ZZ_F8B + 16 * h;
        sp[j] = a.s + t;
    }
    zz_v16f acc[RG][RS];
#pragma unroll
    for (int i = 0; i < RG; i++)
#pragma unroll
        for (int j = 0; j < RS; j++) acc[i][j] = zz_f8_zero();
    struct Block { uint4 w[RG][4], x[RS][4]; float s[RS]; };
    auto load = [&](int b, Block &B) {
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const zz_u4 *from = (const zz_u4 *)(wp[i] + (size_t)b * 4096 + p * 1024);
                const zz_u4 v = NT ? __builtin_nontemporal_load(from) : *from;
                B.w[i][p] = make_uint4(v.x, v.y, v.z, v.w);
            }
#pragma unroll
        for (int j = 0; j < RS; j++) {
#pragma unroll
            for (int p = 0; p < 4; p++) B.x[j][p] = *(const uint4 *)(xp[j] + b * ZZ_F8B + p * 32);
            B.s[j] = sp[j][(size_t)b * rs];
        }
    };
    Block c;
    if (w < nb) load(w, c);
    for (int b = w; b < nb; b += NW) {
        Block n;
        if (PF && b + NW < nb) load(b + NW, n);
        const float wsc = ws[b], wsc2 = wu[b];
        zz_v16f p[RG][RS];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            zz_h8 wf[RG], xf[RS];
#pragma unroll
            for (int i = 0; i < RG; i++) wf[i] = zz_f8_step(c.w[i][k >> 1], k & 1);
#pragma unroll
            for (int j = 0; j < RS; j++) xf[j] = zz_f8_step(c.x[j][k >> 1], k & 1);
#pragma unroll
            for (int i = 0; i < RG; i++)
#pragma unroll
                for (int j = 0; j < RS; j++)
                    p[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[i], xf[j], k ? p[i][j] : zz_f8_zero(), 0, 0, 0);
        }
        float sc[RS], sc2[RS];
#pragma unroll
        for (int j = 0; j < RS; j++) {
            sc[j] = c.s[j] * wsc;
            sc2[j] = G == 2 ? c.s[j] * wsc2 : sc[j];
        }
        if (PF) c = n;
        else if (b + NW < nb) load(b + NW, c);
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int j = 0; j < RS; j++)
#pragma unroll
                for (int k = 0; k < 16; k++) acc[i][j][k] = fmaf(p[i][j][k], k < 8 ? sc[j] : sc2[j], acc[i][j][k]);
    }
    constexpr int TL = RG * RS * 16 * 64;                 // a wave's partial sums
#pragma unroll
    for (int i = 0; i < RG; i++)
#pragma unroll
        for (int j = 0; j < RS; j++)
#pragma unroll
            for (int k = 0; k < 16; k++) part[w * TL + ((i * RS + j) * 16 + k) * 64 + l] = acc[i][j][k];
    __syncthreads();
    constexpr int KQ = GC / 8;
    for (int q = w; q < RG * RS * KQ; q += NW) {          // four columns of a tile a wave
        const int i = q / (RS * KQ), j = q / KQ % RS, k = q % KQ, t = t0 + 32 * j + r;
        if (t >= a.S) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int n = 0; n < NW; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] += part[n * TL + ((i * RS + j) * 16 + 4 * k + e) * 64 + l];
                if constexpr (G == 2) u[e] += part[n * TL + ((i * RS + j) * 16 + 8 + 4 * k + e) * 64 + l];
            }
        const int o = GC * (g0 + i) + 8 * k + 4 * h;
        if constexpr (G) zz_f8_end<G>(a, v, u, o, a.m.O - o, (const T *)a.res + (int64_t)t * a.ldr + o);
        zz_f8_store4((T *)a.y, a.ldy, t, o, a.m.O, v);
    }
}

// 16 bytes (4 bytes) a lane from base + off straight into LDS at lds + 16 (4) * lane, counted
// by vmcnt; no register receives anything. (m0 is named so that nothing of the compiler's is
// kept in it; it warns that it never does.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void zz_dma16(const void *base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void zz_dma4(const void *base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void zz_wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A matrix's scales, one of 64 blocks in each lane: a round takes its own from there by a readlane,
// where a load just before the round's wait for its codes would be waited for with them (512 x 4224 x
// 2816 took 26.4 us with that and takes 25.1). The first is waited for in ready(), behind the first
// blocks' requests (before them 512 x 4224 x 2816 without an epilogue took 20.1 us, behind them 19.7, 512 x
// 65536 x 704 62.3 and 60.8), the later ones where they are made, so that nothing waits for them elsewhere.
struct ZzF8Scales {
    const float *p;
    int nb, base = 0;
    float v;
    __device__ __forceinline__ ZzF8Scales(const float *from, int n) : p(from), nb(n) { load(); }
    __device__ __forceinline__ void load() { v = p[min(base + (int)(threadIdx.x & 63), nb - 1)]; }
    __device__ __forceinline__ void ready() { asm volatile("" : "+v"(v)); }
    __device__ __forceinline__ float of(int b) {           // b ascending, less than nb
        if (b >= base + 64) {
            base = b & ~63;
            load();
            ready();
        }
        return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), b & 63));
    }
};

// Many rows: a workgroup owns a tile of 32*RO*WO matrix rows times 32*RS*WS activation rows.
// KS groups of WO*WS waves take every KS-th block of 128 columns; a wave owns RO x RS tiles of
// 32 x 32. Blocks arrive in LDS NS - 1 rounds ahead without passing registers: matrix codes in
// operand order (a wave's read is one contiguous kilobyte), activation rows as they are, their
// eight 16-byte pieces permuted by (row / 2) % 8 on the way in, so that 16 rows' reads meet 64
// different banks. One barrier a round. Both operands are made f16 as they leave LDS.
//
// At 8192 x 4224 x 2816 (bf16 out) 128 x 128 tiles take 182 us, 1.07 PFLOP/s (the last 64 of 2112
// in quarters; whole they leave a fifth round an eighth full, 191 us); a library f16 product of
// that shape takes 239 (225 in bf16). Of a round's 1.5 us (two workgroups a CU), 0.85 are matrix
// work at 2.4 GHz; the clock is 2.0 to 2.2 GHz under it, and for 16 cycles of matrix work a wave
// issues 3.25 vector operations (two conversions, one fma). Measured beside it and not better
// (191 then): codes through registers (209), 256 x 128 tiles (206), f16 activations in LDS (217),
// a fma phase interleaved with the next tile's products (208), touching later lines for the L2
// (237).
template <int RO, int RS, int WO, int WS, int KS, int NS>
struct ZzF8Async {
    static constexpr int GW = WO * WS, NT = 64 * GW * KS, O = 32 * RO * WO, S = 32 * RS * WS;
    static constexpr int WB = O * 128, XB = S * 128, SB = S * 4 < 256 ? 256 : S * 4, BLOCK = WB + XB + SB;
    static constexpr int STAGE = KS * BLOCK, LDS = NS * STAGE;
    static constexpr int WI = O / 8 / GW, XI = S / 8 / GW, DMA = WI + XI + 1;   // a wave's requests a block
    static_assert(O / 8 % GW == 0 && S / 8 % GW == 0 && SB / 256 <= GW, "whole requests a wave");
    static_assert(LDS >= O * S * 4, "the result's tile");
};

// one tile: the result's rows from t0, the matrix's groups from gt
template <typename T, int G, int RO, int RS, int WO, int WS, int KS, int NS, bool NT, typename A>
__device__ __forceinline__ void zz_fp8_tile(const A &a, char *lds, int gt, int t0) {
    constexpr int GC = zz_f8_gw<G>;
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    const int tid = threadIdx.x, l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int kg = zz_wave_id() / C::GW, w = zz_wave_id() % C::GW, wo = w % WO, ws = w / WO;
    const int g0 = gt + wo * RO, gl = (a.m.O + GC - 1) / GC - 1, last = a.S - 1 - t0, rs = zz_f8_stride<G>(a);
    const float *wsp = a.m.ws + (size_t)(min(g0, gl) / (128 / GC)) * nb, *wup = wsp;
    if constexpr (G == 2) wup += a.wsu;
    const unsigned lb = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds + kg * C::BLOCK;
    // this wave's requests: matrix pieces w*WI .. (4 a group), row octets w*XI .., 64 scales
    const uint8_t *wsrc[C::WI];
#pragma unroll
    for (int i = 0; i < C::WI; i++) {
        const int pc = w * C::WI + i;
        wsrc[i] = a.m.w + (size_t)min(gt + pc / 4, gl) * nb * 4096 + pc % 4 * 1024;
    }
    // (rows by index lie within 2^32 bytes of the first)
    bool by_row = false;
    if constexpr (G) by_row = a.row != nullptr;
    const uint8_t *xsrc = a.q + (by_row ? 0 : (size_t)t0 * nb * ZZ_F8B);
    const float *ssrc = a.s + (by_row ? 0 : t0);
    ZzF8Scales wsl(wsp, nb), wul(wup, nb);
    constexpr int SI = C::SB / 256;
    unsigned xo[C::XI + 1];
#pragma unroll
    for (int i = 0; i < C::XI; i++) xo[i] = min((w * C::XI + i) * 8 + (l >> 3), last);
    xo[C::XI] = min(w % SI * 64 + l, last);
    zz_f8_rows<G>(a, t0, xo);
    const unsigned so = 4 * xo[C::XI];
#pragma unroll
    for (int i = 0; i < C::XI; i++)
        xo[i] = xo[i] * nb * ZZ_F8B + 16 * ((l & 7) ^ ((((w * C::XI + i) & 1) << 2) | (l >> 4)));
    auto fetch = [&](int it, int slot) {
        const int b = min(it * KS + kg, nb - 1);          // behind the last block: its data, not used
        const unsigned d = lb + slot * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::WI; i++) zz_dma16(wsrc[i] + (size_t)b * 4096, l * 16, d + (w * C::WI + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::XI; i++) zz_dma16(xsrc + (size_t)b * ZZ_F8B, xo[i], d + C::WB + (w * C::XI + i) * 1024);
        zz_dma4(ssrc + (size_t)b * rs, so, d + C::WB + C::XB + w % SI * 256);
    };
    zz_v16f acc[RO][RS];
#pragma unroll
    for (int i = 0; i < RO; i++)
#pragma unroll
        for (int j = 0; j < RS; j++) acc[i][j] = zz_f8_zero();
    const int rounds = (nb + KS - 1) / KS;
#pragma unroll
    for (int i = 0; i < NS - 1; i++)
        if (i < rounds) fetch(i, i);
    wsl.ready();
    wul.ready();
    int slot = 0, into = NS - 1;
    for (int it = 0; it < rounds; it++) {
        const int b = it * KS + kg;
        // round it has arrived for this wave; behind the barrier, for all, and the one before it
        // is read
        if (it + NS - 2 < rounds) zz_wait_vm<C::DMA *(NS - 2)>();
        else zz_wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (it + NS - 1 < rounds) fetch(it + NS - 1, into);
        const char *d = lds + slot * C::STAGE + kg * C::BLOCK;
        slot = slot + 1 == NS ? 0 : slot + 1;
        into = into + 1 == NS ? 0 : into + 1;
        if (KS > 1 && b >= nb) continue;
        const float wsc = wsl.of(b), wsc2 = G == 2 ? wul.of(b) : wsc;
        float sc[RS], sc2[RS];
#pragma unroll
        for (int j = 0; j < RS; j++) {
            const float xsc = *(const float *)(d + C::WB + C::XB + 4 * ((ws * RS + j) * 32 + r));
            sc[j] = xsc * wsc;
            sc2[j] = G == 2 ? xsc * wsc2 : sc[j];
        }
        zz_v16f p[RO][RS];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint4 wv[RO], xv[RS];
#pragma unroll
            for (int i = 0; i < RO; i++) wv[i] = *(const uint4 *)(d + ((wo * RO + i) * 4 + k) * 1024 + l * 16);
#pragma unroll
            for (int j = 0; j < RS; j++)
                xv[j] = *(const uint4 *)(d + C::WB + ((ws * RS + j) * 32 + r) * 128 + 16 * ((2 * k + h) ^ ((r >> 1) & 7)));
#pragma unroll
            for (int e = 0; e < 2; e++) {
                zz_h8 wf[RO], xf[RS];
#pragma unroll
                for (int i = 0; i < RO; i++) wf[i] = zz_f8_step(wv[i], e);
#pragma unroll
                for (int j = 0; j < RS; j++) xf[j] = zz_f8_step(xv[j], e);
#pragma unroll
                for (int i = 0; i < RO; i++)
#pragma unroll
                    for (int j = 0; j < RS; j++)
                        p[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[i], xf[j], k || e ? p[i][j] : zz_f8_zero(), 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < RO; i++)
#pragma unroll
            for (int j = 0; j < RS; j++)
#pragma unroll
                for (int k = 0; k < 16; k++) acc[i][j][k] = fmaf(p[i][j][k], k < 8 ? sc[j] : sc2[j], acc[i][j][k]);
    }
    // The tile goes through LDS, [row][column] in 16-byte pieces (a row's pieces permuted by the
    // row, for the banks), where the K groups are added in their order; then whole lines leave.
    float *tile = (float *)lds;
    auto place = [&](int t, int o) { return tile + t * C::O + 4 * ((((o >> 2) ^ t) & 7) | ((o >> 2) & ~7)); };
#pragma unroll
    for (int g = 0; g < KS; g++) {
        __syncthreads();                                  // the last block, or the group before, is read
        if (kg == g)
#pragma unroll
            for (int i = 0; i < RO; i++)
#pragma unroll
                for (int j = 0; j < RS; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float4 *q = (float4 *)place((ws * RS + j) * 32 + r, (wo * RO + i) * 32 + 8 * k + 4 * h);
                        float4 v = make_float4(acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]);
                        if (g) {
                            const float4 u = *q;
                            v = make_float4(u.x + v.x, u.y + v.y, u.z + v.z, u.w + v.w);
                        }
                        *q = v;
                    }
    }
    __syncthreads();
    constexpr int E = 16 / sizeof(T), RL = C::O / 32 * GC / E;      // elements a lane stores, lanes a row
    for (int i = tid; i < C::S * RL; i += C::NT) {
        const int t = i / RL, o = (i % RL) * E, from = o / GC * 32 + o % GC, col = gt * GC + o;
        if (t > last) break;
        float v[E], u[E];
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            *(float4 *)(v + e) = *(const float4 *)place(t, from + e);
            if constexpr (G == 2) *(float4 *)(u + e) = *(const float4 *)place(t, from + 16 + e);
        }
        if constexpr (G) zz_f8_end<G>(a, v, u, col, a.m.O - col, (const T *)a.res + (int64_t)(t0 + t) * a.ldr + col);
        zz_f8_store<NT>((T *)a.y + (int64_t)(t0 + t) * a.ldy + col, v, a.m.O - col);
    }
}

// Tile id's place: panels of PW row tiles, whose columns the XCDs go through side by side.
__device__ __forceinline__ void zz_fp8_at(int id, int OT, int ST, int *ot, int *st) {
    constexpr int PW = 8;
    const int pan = id / (OT * PW), in = id - pan * OT * PW, pw = min(PW, ST - pan * PW);
    *ot = in / pw;
    *st = pan * PW + in % pw;
}
