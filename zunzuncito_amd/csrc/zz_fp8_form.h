// zz_fp8_form.h -- which form a product of e4m3 rows takes (include/zz_fp8.h): rules on sizes, host
// code without HIP, so that they can be looked at without a device too.
#pragma once
#include <math.h>
#include <stdint.h>

// An output of at least this many bytes, a quarter of the 256 MB cache in front of memory, is
// stored past it: who reads it next finds little of it there, and its dirty lines would be
// written back under the next kernels' reads.
#define ZZ_NT_BYTES ((int64_t)64 << 20)

// Forms by number; their kernels are in zz_fp8_mma.hip (launch_mm) and zz_fp8_ep.h (launch_ep). 0 to 2
// for few rows, 3 to 10 tiles on the f16 instructions, 11 to 13 on the 8-bit ones. A choice is of all
// that a plain product has, of what one with an epilogue has, or of that and the 8-bit tiles.
#define ZZ_F8_FORMS_PLAIN 0
#define ZZ_F8_FORMS_EP    1
#define ZZ_F8_FORMS_8BIT  2

// Which form for `tables` products of S rows each: the one that is expected to take the shortest. A
// form's workgroups go round by round through the 256 CUs, `per` of them on a CU at once; a round with
// k workgroups on the busiest CU takes fix[k-1] + slope[k-1] * (blocks that a K group runs)
// microseconds. A form with `parts` runs what is over a multiple of 256 tiles in that many parts each, if these are at most
// one a CU: 2.9 + 0.49 * blocks after a full round, or less beside workgroups that are there
// (`busy`: fixed, a block, a block with a part on each CU). Fitted to 114 shapes (O 704 to 65536,
// I 256 to 8192, S 1 to 8192) with an rms error of 6 to 17 %. Over them the choice lies 2 % behind
// the best form of each, and up to 17 %. Any one form for all loses far more: 32 x 32 in sixteen
// groups and 128 x 128 take 4.8 and 25.6 us for 1 x 4224 x 2816, 295 and 109 for 4096 rows; without the
// parts 4096 x 4224 x 2816 takes 107 us where it takes 95, 1000 x 4224 x 2816 36 for 30.
// The model has no bandwidth in it and holds for what it was fitted to. For few rows of matrices
// past the caches its times lie below what their bytes take (262144 x 4096: 131 us, where a read at
// 7.1 TB/s takes 151), and from about 3700 columns on it prefers the third form, whose loads go
// through the caches: 1 row of 262144 x 4096 180 us (6.0 TB/s), of 128256 x 7168 152 (6.1), of 18432
// x 7168 30 (4.4), where the second form's past the caches reaches 6.9 at 262144 x 2816.
struct ZzF8Form { int o, s, ks, per; float fix[4], slope[4]; int parts; float busy[3]; };
static const ZzF8Form zz_f8_forms[] = {
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
    // zz_fp8_wide.h's, from 512 and 2816 columns with one to `per` workgroups on each CU: over 188 shapes (O 704
    // to 32768, I 300 to 8192, S 1 to 8192) the rms error is 17 to 21 %, most of it times that are too long,
    // and the choice among these and the first six lies 2.7 % behind the best, and up to 31 %; over the same
    // shapes, with an epilogue, the choice among the others 1.7 %, and up to 14 %
    {64, 64, 1, 4, {4.6f, 5.6f, 6.5f, 6.9f}, {0.41f, 0.45f, 0.48f, 0.62f}},
    {128, 64, 1, 3, {5.1f, 6.6f, 7.6f}, {0.46f, 0.58f, 0.81f}},
    {128, 128, 1, 2, {7.8f, 9.2f}, {0.63f, 0.93f}},
};
static inline int zz_fp8_form(int O, int S, int tables, int nb, int of) {
    int best = 0;
    float least = INFINITY;
    // up to 32 rows the first three: the others' tiles are half empty
    for (int v = 0; v < (S <= 32 ? 3 : of == ZZ_F8_FORMS_8BIT ? 14 : 11); v++) {
        const ZzF8Form &f = zz_f8_forms[v];
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

// The form for P rows of m matrices, `per` each on average, O packed rows, nb blocks: zz_fp8_form's
// choice, but for tables of several from 1024 workgroups of the few-row form on. How the rows are spread
// is not known here; even, mildly uneven, by Zipf's law (1.1) and over 8 experts alone were measured, 32
// tables of 2 to 512 experts, 1 to 512 rows an expert. Figures are of bf16 results, f32's within 3 %.
// On the f16 instructions up to 2 rows an expert the second form (128 experts of 2 x 704 x 2816, 2 rows
// each: 77 us, the fourth 92), up to 32 the fourth, 64 x 32 tiles (8 rows each, and by Zipf's law: 93 and 90 us,
// the second 85 and 89; 32 rows: 108 and 128, the second 136 and 175, 64 x 128 tiles 148 and 166): 1.5 to 3 %
// behind the best form of each, 11 % where 8 experts have all rows, and up to 1.9 times as long there
// (of 256, 2048 x 768, 32 rows each on average: 76 us, 128 x 128 tiles 44).
// On the 8-bit ones from 2^19 packed results on 128 x 64 tiles at least, whatever an expert's rows (128
// experts of 4096 x 1024, by Zipf's law 1, 8, 32 rows each: 39, 91, 110 us, the second form 49, 112, 204; of
// 2 x 704 x 2816, 4 rows each, 91 and 79), below that the second: 3 to 4 % behind the best of each.
static inline int zz_f8_ep_form(int O, int P, int per, int m, int nb, bool eight) {
    const int v = zz_fp8_form(O, per, m, nb, eight ? ZZ_F8_FORMS_8BIT : ZZ_F8_FORMS_EP);
    if (m == 1) return v;
    if (eight && (int64_t)P * O >= 1 << 19) return v > 12 ? v : 12;
    if (per > 32 || (int64_t)m * ((O + 31) / 32) <= 1024) return v;
    return eight || per <= 2 ? 1 : 3;
}

// The most row tiles of `ts` rows that P rows of E matrices can make; one matrix without a table
static inline int64_t zz_f8_ep_tiles(int P, int E, bool table, int ts) {
    const int64_t m = table ? (E < P ? E : P) : 1;
    return (P + m * (ts - 1)) / ts;
}

// whether a launch in one dimension holds n workgroups of `threads`
static inline bool zz_f8_fits(int64_t n, int threads) { return n * threads <= 0xffffffffll; }

// whether there is a form whose launch holds P rows of O packed rows: the largest tiles, 128 x 128 by 256
static inline bool zz_f8_ep_fits(int O, int P, int E, bool table) {
    return zz_f8_fits((zz_f8_ep_tiles(P, E, table, 128) * ((O + 127) / 128) + 7) / 8 * 8, 256);
}

// The kernel of a product with an epilogue: P rows of a table of E matrices (`table`; else one), O packed
// rows and I columns each. A form, but 14 to 16 the second form's for matrices past the caches, which
// are read past them too, as zz_fp8_mma.hip's: of several matrices by four waves a workgroup, as the second
// form's (128 pairs to 8 of 128 experts, 1408 x 2816: 11.9 us, by eight 17.5), of one for up to 8 rows, and for more.
static inline int zz_f8_ep_kernel(int O, int I, int P, int E, bool table, bool eight) {
    // the matrices that can have rows, and each one's rows, were they spread evenly
    const int m = table ? (E < P ? E : P) : 1, per = (P + m - 1) / m;
    const int v = zz_f8_ep_form(O, P, per, m, (I + 127) / 128, eight);
    if (v != 1 || per > 32 || (int64_t)m * O * I < ZZ_NT_BYTES) return v;
    return m > 1 ? 14 : per <= 8 ? 15 : 16;
}
