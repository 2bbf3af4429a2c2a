// zz_fp8_mma.hip -- products of e4m3 rows with resident e4m3 matrices on the matrix cores
// (include/zz_fp8.h).
//
//   y[s][o] = sum_b xs[b][s] * ws[o/128][b] * sum_{k in block b} xq[s][k] wq[o][k]
// The codes are multiplied as f16, which holds every e4m3 value: the products are exact and
// the matrix core adds them up in f32. The 8-bit instructions do not: they align 16 products
// to the largest and keep 13 bits behind it (2^-14 beside 1 is lost within 16 neighbours and
// kept between them, measured), 1.5e-5 off in the 2-norm over normally distributed codes and
// 1e-4 of the terms' magnitude at worst, where the f16 form is 1e-8 and 2e-7 off. They would
// run at twice the rate (8192^3 in a library 2.7 PFLOP/s, in f16 1.35). Results in bf16, whose own
// rounding is a hundred times as large, would bear them, but take the same form. bf16 holds
// every code too, and its library product is faster (1.48): not tried.
//
// A block of 128 columns is eight v_mfma_f32_32x32x16_f16 of 32 matrix rows times 32
// activation rows; each of the 16 results a lane then enters the f32 accumulator by one fma
// with the two scales' product. Lane 32h + r holds activation row r and the matrix rows
// 8k + 4h .. + 3 (k = 0..3) of the group, so a lane needs one row scale and a group one matrix
// scale. (The 16x16x32 form leaves 3 of 4 issue slots to the conversions and fma's beside it,
// this one 7 of 8: with 3 vector operations for each 16 cycles of matrix work, as here, 24 and
// 19 cycles were measured.)
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

// Few rows: a workgroup per RG groups of 32 matrix rows and RS tiles of 32 activation rows;
// its NW waves take every NW-th block, straight from memory into registers (PF: the next one's
// codes requested before the current one is multiplied), and meet in LDS, where the partial
// sums are added in the waves' order. Rows behind the last one are read as the last one, and
// not stored. NT: the matrix is read once and does not stay in the caches: 3 rows against
// 262144 x 2816 in 104 us, 7.1 TB/s, instead of 120.
template <typename T, int RG, int RS, int NW, bool PF, bool NT>
__global__ __launch_bounds__(64 * NW) void zz_fp8_few_kernel(ZzF8Mm a) {
    extern __shared__ __attribute__((aligned(16))) float part[];     // [NW][RG][RS][16][64]
    const int tid = threadIdx.x, w = zz_wave_id(), l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int g0 = blockIdx.x * RG, gl = (a.m.O + 31) / 32 - 1, t0 = blockIdx.y * 32 * RS;
    const uint8_t *wp[RG], *xp[RS];
    const float *ws = a.m.ws + (size_t)(g0 / 4) * nb, *sp[RS];
#pragma unroll
    for (int i = 0; i < RG; i++) wp[i] = a.m.w + (size_t)min(g0 + i, gl) * nb * 4096 + l * 16;
#pragma unroll
    for (int j = 0; j < RS; j++) {
        const int t = min(t0 + 32 * j + r, a.S - 1);
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
            B.s[j] = sp[j][(size_t)b * a.S];
        }
    };
    Block c;
    if (w < nb) load(w, c);
    for (int b = w; b < nb; b += NW) {
        Block n;
        if (PF && b + NW < nb) load(b + NW, n);
        const float wsc = ws[b];
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
        float sc[RS];
#pragma unroll
        for (int j = 0; j < RS; j++) sc[j] = c.s[j] * wsc;
        if (PF) c = n;
        else if (b + NW < nb) load(b + NW, c);
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
            for (int j = 0; j < RS; j++)
#pragma unroll
                for (int k = 0; k < 16; k++) acc[i][j][k] = fmaf(p[i][j][k], sc[j], acc[i][j][k]);
    }
    constexpr int TL = RG * RS * 16 * 64;                 // a wave's partial sums
#pragma unroll
    for (int i = 0; i < RG; i++)
#pragma unroll
        for (int j = 0; j < RS; j++)
#pragma unroll
            for (int k = 0; k < 16; k++) part[w * TL + ((i * RS + j) * 16 + k) * 64 + l] = acc[i][j][k];
    __syncthreads();
    for (int q = w; q < RG * RS * 4; q += NW) {           // four matrix rows of a tile a wave
        const int i = q / (RS * 4), j = q / 4 % RS, k = q % 4, t = t0 + 32 * j + r;
        if (t >= a.S) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int u = 0; u < NW; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += part[u * TL + ((i * RS + j) * 16 + 4 * k + e) * 64 + l];
        zz_f8_store4((T *)a.y, a.ldy, t, 32 * (g0 + i) + 8 * k + 4 * h, a.m.O, v);
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

// one tile: the result's rows from t0 and columns from 32 * gt
template <typename T, int RO, int RS, int WO, int WS, int KS, int NS, bool NT>
__device__ __forceinline__ void zz_fp8_tile(const ZzF8Mm &a, char *lds, int gt, int t0) {
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    const int tid = threadIdx.x, l = tid & 63, r = l & 31, h = l >> 5, nb = a.nb;
    const int kg = zz_wave_id() / C::GW, w = zz_wave_id() % C::GW, wo = w % WO, ws = w / WO;
    const int g0 = gt + wo * RO, gl = (a.m.O + 31) / 32 - 1, last = a.S - 1 - t0;
    const float *wsp = a.m.ws + (size_t)(min(g0, gl) / 4) * nb;
    const unsigned lb = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds + kg * C::BLOCK;
    // this wave's requests: matrix pieces w*WI .. (4 a group), row octets w*XI .., 64 scales
    const uint8_t *wsrc[C::WI];
#pragma unroll
    for (int i = 0; i < C::WI; i++) {
        const int pc = w * C::WI + i;
        wsrc[i] = a.m.w + (size_t)min(gt + pc / 4, gl) * nb * 4096 + pc % 4 * 1024;
    }
    const uint8_t *xsrc = a.q + (size_t)t0 * nb * ZZ_F8B;
    const float *ssrc = a.s + t0;
    unsigned xo[C::XI];
#pragma unroll
    for (int i = 0; i < C::XI; i++)
        xo[i] = (unsigned)min((w * C::XI + i) * 8 + (l >> 3), last) * nb * ZZ_F8B +
                16 * ((l & 7) ^ ((((w * C::XI + i) & 1) << 2) | (l >> 4)));
    constexpr int SI = C::SB / 256;
    const unsigned so = 4 * (unsigned)min(w % SI * 64 + l, last);
    auto fetch = [&](int it, int slot) {
        const int b = min(it * KS + kg, nb - 1);          // behind the last block: its data, not used
        const unsigned d = lb + slot * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::WI; i++) zz_dma16(wsrc[i] + (size_t)b * 4096, l * 16, d + (w * C::WI + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::XI; i++) zz_dma16(xsrc + (size_t)b * ZZ_F8B, xo[i], d + C::WB + (w * C::XI + i) * 1024);
        zz_dma4(ssrc + (size_t)b * a.S, so, d + C::WB + C::XB + w % SI * 256);
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
    int slot = 0, into = NS - 1;
    for (int it = 0; it < rounds; it++) {
        const int b = it * KS + kg;
        const float wsc = b < nb ? wsp[b] : 0.0f;
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
        float sc[RS];
#pragma unroll
        for (int j = 0; j < RS; j++) sc[j] = *(const float *)(d + C::WB + C::XB + 4 * ((ws * RS + j) * 32 + r)) * wsc;
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
                for (int k = 0; k < 16; k++) acc[i][j][k] = fmaf(p[i][j][k], sc[j], acc[i][j][k]);
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
    constexpr int E = 16 / sizeof(T), RL = C::O / E;      // elements a lane stores, lanes a row
    for (int i = tid; i < C::S * RL; i += C::NT) {
        const int t = i / RL, o = (i % RL) * E;
        if (t > last) break;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; e += 4) *(float4 *)(v + e) = *(const float4 *)place(t, o + e);
        zz_f8_store<NT>((T *)a.y + (int64_t)(t0 + t) * a.ldy + gt * 32 + o, v, a.m.O - gt * 32 - o);
    }
}

// Tile id's place: panels of PW row tiles, whose columns the XCDs go through side by side.
__device__ __forceinline__ void zz_fp8_at(int id, int OT, int ST, int *ot, int *st) {
    constexpr int PW = 8;
    const int pan = id / (OT * PW), in = id - pan * OT * PW, pw = min(PW, ST - pan * PW);
    *ot = in / pw;
    *st = pan * PW + in % pw;
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
    zz_fp8_tile<T, RO, RS, WO, WS, KS, NS, false>(a, lds, ot * C::O / 32, st * C::S);
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
        zz_fp8_tile<T, RO, RS, 2, 2, 1, 2, NT>(a, lds, ot * 2 * RO, st * 64 * RS);
    } else {
        const int part = (x - 8 * g) % (RO * RS);
        zz_fp8_at(whole + (x - 8 * g) / (RO * RS), OT, ST, &ot, &st);
        const int gt = (ot * RO + part % RO) * 2, t0 = (st * RS + part / RO) * 64;
        if (gt * 32 < a.m.O && t0 < a.S) zz_fp8_tile<T, 1, 1, 2, 2, 1, 3, NT>(a, lds, gt, t0);
    }
}

// one 16-byte piece of the packed layout per thread
__global__ __launch_bounds__(256) void zz_fp8_pack_kernel(const uint8_t *src, int O, int I, int nb, uint8_t *dst,
                                                          int64_t n) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    const int l = (int)(p & 63), pc = (int)(p >> 6) & 3;
    const int64_t gb = p >> 8, g = gb / nb;
    const int b = (int)(gb - g * nb), k = b * ZZ_F8B + 32 * pc + 16 * (l >> 5);
    const int64_t row = g * 32 + (l & 31);
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

int zz_launch_fp8_pack(const uint8_t *codes, int O, int I, uint8_t *dst, hipStream_t st) {
    const int nb = zz_f8_nb(I);
    const int64_t n = (int64_t)((O + 31) / 32) * nb * 256;
    hipLaunchKernelGGL(zz_fp8_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, codes, O, I, nb, dst, n);
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
};
static int mm_plan(int O, int S, int nb) {
    int best = 0;
    float least = INFINITY;
    // up to 32 rows the first three: the others' tiles are half empty
    for (int v = 0; v < (S <= 32 ? 3 : (int)(sizeof mm_forms / sizeof *mm_forms)); v++) {
        const ZzF8Form &f = mm_forms[v];
        int64_t n = (int64_t)((O + f.o - 1) / f.o) * ((S + f.s - 1) / f.s);
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
    const int v = mm_plan(a.m.O, a.S, a.nb);
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
