// zz_beam.hip -- beam search's step (include/zz_beam.h).
//
//   total(w, t) = score[w] + ((L[w][t] - m[w]) - log(sum_t exp(L[w][t] - m[w]))), m the maximum
// Within a row totals go by the logit, so a row's W best are found on the logits alone, as
// 64-bit keys (order-preserving bits of the logit, then the lower token), and the sum of
// exponentials belongs to the same pass over the data; within a chunk it is summed in f32 (up to
// 32 terms a thread, then the wave's and the workgroup's), from there on in double. Two launches:
//   zz_beam_part_kernel   a workgroup per (row, chunk of the vocabulary): the chunk's W
//                         largest keys in order, its maximum and sum of exponentials
//   zz_beam_merge_kernel  a workgroup per sequence: a wave per beam joins the chunks' lists
//                         and sums (in double), and finds its totals' places among all
// or, for a small vocabulary, one: zz_beam_small_kernel, whose waves make their beams' lists
// themselves. A step of 16 sequences of 8 beams over 262144 f32 logits takes 32 us, 134 MB at
// 4.2 TB/s, 26 us of it in the first launch at 5.2 TB/s; in bf16 29 us. There it is the chain of
// a chunk's steps, at five workgroups a CU, and neither bytes nor instructions: without the
// instructions that make NaN harmless it took as long.
#include "zz_common.h"
#include "zz_kernels.h"
#include "zz_fp8_dev.h"
#include "../../include/zz_beam.h"

#include <math.h>

#define ZZ_FAIL(...)               \
    do {                           \
        zz_set_error(__VA_ARGS__); \
        return 0;                  \
    } while (0)

typedef unsigned long long zz_u64;

// order-preserving bits of a float that is no NaN
__device__ __forceinline__ unsigned zz_ord32(float f) {
    const unsigned u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float zz_unord32(unsigned u) {
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ zz_u64 zz_ord64(double d) {
    const zz_u64 u = (zz_u64)__double_as_longlong(d);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double zz_unord64(zz_u64 u) {
    return __longlong_as_double((long long)((u >> 63) ? (u & 0x7fffffffffffffffull) : ~u));
}
// a candidate: the larger key is the better one; 0 is none (no float's bits order to 0)
// (minus zero is zero)
__device__ __forceinline__ zz_u64 zz_beam_key(float v, int t) {
    return ((zz_u64)zz_ord32(v + 0.0f) << 32) | (0xffffffffu - (unsigned)t);
}

// lane q's (q wave-uniform)
__device__ __forceinline__ unsigned zz_lane_u32(unsigned v, int q) {
    return (unsigned)__builtin_amdgcn_readlane((int)v, q);
}
__device__ __forceinline__ zz_u64 zz_lane_u64(zz_u64 v, int q) {
    return ((zz_u64)zz_lane_u32((unsigned)(v >> 32), q) << 32) | zz_lane_u32((unsigned)v, q);
}

// the wave's largest key: the upper words first, the lower ones only where several lanes share
// the upper word (equal logits)
__device__ __forceinline__ zz_u64 zz_wave_max64(zz_u64 v) {
    const unsigned hi = (unsigned)(v >> 32), lo = (unsigned)v;
    auto mx = [](unsigned a, unsigned b) { return a > b ? a : b; };
    const unsigned H = zz_group_reduce<64>(hi, mx);
    const zz_u64 at = __ballot(hi == H);
    unsigned L;
    if (__popcll(at) == 1) L = zz_lane_u32(lo, __ffsll((long long)at) - 1);
    else L = zz_group_reduce<64>(hi == H ? lo : 0u, mx);
    return ((zz_u64)H << 32) | L;
}

struct ZzBeamArgs {
    const void *logits;
    int64_t ldl;
    int N, W, V, chunks, eos, pad;
    const float *score;
    const uint8_t *done;            // may be null
    float *score_out;
    int *parent, *token;
    uint8_t *done_out;              // may be null
    zz_u64 *ws;                     // [N*W][chunks][W + 1]: keys, then (maximum, sum)
};

// what a wave's lanes stored in LDS, read by the others
__device__ __forceinline__ void zz_wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A thread's share of a row: NV pieces of 16 bytes, pieces first, first + step, ... counted from
// the row's first token: the sum's order does not depend on where the row lies, so equal rows
// have equal totals. A row of an odd vocabulary begins at any multiple of its element; the loads
// need no more. A piece across the row's end goes element by element.
template <typename T, int NV>
struct ZzBeamShare {
    static constexpr int VE = 16 / sizeof(T), NE = NV * VE;
    float v[NE];
    int V, first, step;

    __device__ __forceinline__ ZzBeamShare(const T *L, int V_, int first_, int step_) : V(V_), first(first_), step(step_) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = (first + i * step) * VE;
            if (e + VE <= V) {
                unsigned u[4];
                __builtin_memcpy(u, L + e, 16);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (VE == 4) {
                        v[4 * i + j] = __uint_as_float(u[j]);
                    } else {
                        v[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
                        v[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < VE; j++) v[VE * i + j] = e + j < V ? zz_f32_of(L[e + j]) : NAN;
            }
        }
    }
    // the token of element k, or -1 where it lies outside the row
    __device__ __forceinline__ int tok(int k) const {
        const int t = (first + k / VE * step) * VE + k % VE;
        return t < V ? t : -1;
    }
    __device__ __forceinline__ float max() {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NE; k++) {
            v[k] = fmaxf(v[k], -INFINITY);               // a NaN counts as minus infinity
            m = fmaxf(m, v[k]);
        }
        return m;
    }
    // the sum of exp(v - m)
    __device__ __forceinline__ float sum(float m) const {
        float s = 0.0f;
        if (fabsf(m) < 16384.0f) {
            // 2^(v log2(e) - c), c = m log2(e) rounded; what c's rounding left is a common factor
            const float c = m * ZZ_LOG2E, off = fmaf(m, ZZ_LOG2E, -c);
#pragma unroll
            for (int k = 0; k < NE; k++) s += __builtin_amdgcn_exp2f(fmaf(v[k], ZZ_LOG2E, -c));
            s *= __builtin_amdgcn_exp2f(-off);
        } else if (fabsf(m) != INFINITY) {
#pragma unroll
            for (int k = 0; k < NE; k++) s += __builtin_amdgcn_exp2f((v[k] - m) * ZZ_LOG2E);
        } else {
            // the infinite logits share the probability; at minus infinity the sum is not used
#pragma unroll
            for (int k = 0; k < NE; k++) s += v[k] == m ? 1.0f : 0.0f;
        }
        return s;
    }
    // the wave's keys of logits that reach the line, to cand while they are up to 64; their number
    __device__ __forceinline__ int gather(float line, zz_u64 *cand) const {
        int total = 0;
        auto walk = [&](auto in) {
#pragma unroll
            for (int k = 0; k < NE; k++) {
                const bool is = in(k);
                const zz_u64 at = __ballot(is);
                if (at) {
                    const int o = total + __builtin_amdgcn_mbcnt_hi((unsigned)(at >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)at, 0));
                    if (is && o < 64) cand[o] = zz_beam_key(v[k], tok(k));
                    total += __popcll(at);
                }
            }
        };
        if (line != -INFINITY) walk([&](int k) { return v[k] >= line; });
        else walk([&](int k) { return tok(k) >= 0; });   // what lies outside the row is there too
        return total;
    }
    // the wave's W largest keys, a round each: for more than 64 at the line
    __device__ __forceinline__ void rounds(int W, zz_u64 *best) const {
        zz_u64 prev = ~0ull;
        for (int k = 0; k < W; k++) {
            zz_u64 b = 0;
#pragma unroll
            for (int j = 0; j < NE; j++) {
                const int t = tok(j);
                const zz_u64 key = t < 0 ? 0 : zz_beam_key(v[j], t);
                if (key < prev && key > b) b = key;
            }
            prev = zz_wave_max64(b);
            if ((threadIdx.x & 63) == 0) best[k] = prev;
        }
    }
};

// The W-th largest of the lanes' lm, m the largest. Rounds of a wave's maximum find it for up to
// 8 beams (a step of 1 sequence over 4096 logits, 4 beams: 6.3 us against 6.6); beyond, it is the
// least of those with fewer than W above them, counted (16 beams: 9.7 us against 10.7).
// lms: 64 floats of LDS.
__device__ __forceinline__ float zz_beam_line(float lm, float m, int W, float *lms) {
    const int l = threadIdx.x & 63;
    float line = m;
    if (W <= 8) {
        for (int k = 1; k < W; k++) {
            const zz_u64 at = __ballot(lm == line);
            if (l == __ffsll((long long)at) - 1) lm = -INFINITY;
            line = zz_wave_max(lm);
        }
        return line;
    }
    lms[l] = lm;
    zz_wave_lds();
    int above = 0;
#pragma unroll
    for (int j = 0; j < 64; j++) above += lms[j] > lm;
    line = -zz_wave_max(above < W ? -lm : -INFINITY);
    zz_wave_lds();
    return line;
}

// The place of a lane's key among n <= 64 distinct ones, one a lane and 0 beyond: the number of
// better ones. keys: 64 of LDS, which then hold them.
__device__ __forceinline__ int zz_beam_place(zz_u64 key, int n, zz_u64 *keys) {
    keys[threadIdx.x & 63] = key;
    zz_wave_lds();
    int rank = 0;
    for (int j = 0; j < n; j += 8)
#pragma unroll
        for (int u = 0; u < 8; u++) rank += keys[j + u] > key;
    zz_wave_lds();
    return rank;
}

__device__ __forceinline__ zz_u64 zz_beam_sum(float m, float s) { return ((zz_u64)__float_as_uint(s) << 32) | __float_as_uint(m); }

// A workgroup per (chunk, row); its waves' pieces are interleaved. At least W logits reach the
// W-th largest of 64 groups' maxima (a lane of each wave is a group), and the W best do: a few
// more than W, unless many are equal. One wave finds that line while the others sum, and ranks
// what all gathered.
template <typename T, int NV>
__global__ __launch_bounds__(256) void zz_beam_part_kernel(ZzBeamArgs a) {
    __shared__ zz_u64 cand[4][64];
    __shared__ float lms[256], wsum[4], lines;
    __shared__ int count[4];
    const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x, l = tid & 63, w = zz_wave_id(), W = a.W;
    if (a.done && a.done[row]) return;
    ZzBeamShare<T, NV> x((const T *)a.logits + row * a.ldl, a.V, ch * NV * 256 + tid, 256);
    lms[tid] = x.max();
    __syncthreads();
    const float lm = fmaxf(fmaxf(lms[l], lms[64 + l]), fmaxf(lms[128 + l], lms[192 + l])), m = zz_wave_max(lm);
    if (w == 0) {
        const float line = zz_beam_line(lm, m, W, (float *)cand[0]);
        if (l == 0) lines = line;
    }
    const float s = zz_wave_sum(x.sum(m));
    if (l == 0) wsum[w] = s;
    __syncthreads();
    int n = x.gather(lines, cand[w]);
    if (l == 0) count[w] = n;
    __syncthreads();
    int c0 = count[0], c1 = count[1], c2 = count[2], c3 = count[3];
    if (c0 + c1 + c2 + c3 > 64) {
        x.rounds(W, cand[w]);
        __syncthreads();
        c0 = c1 = c2 = c3 = W;
    }
    if (w != 0) return;
    n = c0 + c1 + c2 + c3;
    const int q = (l >= c0) + (l >= c0 + c1) + (l >= c0 + c1 + c2);
    const int before = (q > 0 ? c0 : 0) + (q > 1 ? c1 : 0) + (q > 2 ? c2 : 0);
    const zz_u64 key = l < n ? cand[q][l - before] : 0;
    zz_wave_lds();
    const int rank = zz_beam_place(key, n, cand[0]);
    zz_u64 *out = a.ws + ((size_t)row * a.chunks + ch) * (W + 1);
    if (key && rank < W) out[rank] = key;
    if (l < W && l >= __popcll(__ballot(key != 0))) out[l] = 0;
    if (l == 0) out[W] = zz_beam_sum(m, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]));
}

// The W best of n <= 64 lists of distinct keys (list i at p + i * stride: W keys in order, 0
// behind the last), by one wave: lane k < W receives the k-th, 0 if there are fewer. Serial rounds
// of a wave's maximum cost their latency W times over; so a key's place is counted, as the number
// of better ones, among as many of the lists' first keys as the wave has lanes. Where these are
// not all keys, the W-th of them (by its logit) is a bound that the W best reach, and few others
// do; only if more than 64 reach it, rounds decide. cand: 64 keys of LDS of the wave's own.
__device__ __forceinline__ zz_u64 zz_beam_best(const zz_u64 *p, int stride, int n, int W, zz_u64 *cand) {
    const int l = threadIdx.x & 63;
    if (n == 1) return l < W ? p[l] : 0;
    // 64 / n keys of each, down to a power of two, or one that holds W
    const int sh = min(__builtin_clz(n - 1) - 26, W > 1 ? 32 - __builtin_clz(W - 1) : 0);
    const int i = l >> sh, k = l & ((1 << sh) - 1);
    zz_u64 key = i < n && k < W ? p[i * stride + k] : 0;
    int m = n << sh;
    if (1 << sh < W) {
        const unsigned hi = (unsigned)(key >> 32);
        unsigned *his = (unsigned *)cand;
        his[l] = hi;
        zz_wave_lds();
        int above = 0;
#pragma unroll
        for (int j = 0; j < 64; j++) above += his[j] > hi;
        const unsigned line = zz_group_reduce<64>(above < W ? ~hi : 0u, [](unsigned x, unsigned y) { return x > y ? x : y; });
        const zz_u64 bar = (zz_u64)~line << 32;
        zz_wave_lds();
        cand[l] = 0;
        m = bar ? 0 : 65;
        for (int q = 0; q < W && m <= 64; q++) {
            const zz_u64 mine = l < n ? p[l * stride + q] : 0;
            const zz_u64 in = __ballot(mine >= bar);
            if (!in) break;
            const int o = m + __builtin_amdgcn_mbcnt_hi((unsigned)(in >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)in, 0));
            if (mine >= bar && o < 64) cand[o] = mine;
            m += __popcll(in);
        }
        if (m > 64) {
            int first = 0;
            zz_u64 head = l < n ? p[l * stride] : 0, got = 0;
            for (int q = 0; q < W; q++) {
                const zz_u64 b = zz_wave_max64(head);
                if (l == q) got = b;
                if (head == b && b) {
                    first++;
                    head = first < W ? p[l * stride + first] : 0;
                }
            }
            return got;
        }
        zz_wave_lds();
        key = cand[l];
    }
    const int rank = zz_beam_place(key, m, cand);
    cand[l] = 0;
    zz_wave_lds();
    if (key) cand[rank] = key;
    zz_wave_lds();
    return cand[l];
}

// What a sequence's workgroup picks from, in LDS.
struct ZzBeamPick {
    zz_u64 tot[ZZ_BEAM_MAXW][ZZ_BEAM_MAXW];              // a beam's best totals in order, 0: none
    zz_u64 cand[ZZ_BEAM_MAXW][64];                       // a wave's own
};

// A wave per beam: `mine`, its row's C lists with their sums, to the row's W best totals, and
// these to their places among the sequence's.
__device__ __forceinline__ void zz_beam_finish(const ZzBeamArgs &a, ZzBeamPick &P, const zz_u64 *mine, int C, bool done,
                                               float c) {
    const int w = zz_wave_id(), l = threadIdx.x & 63, W = a.W;
    if (c != c) c = -INFINITY;
    zz_u64 tot = 0;
    int tok = a.pad;
    if (done) {
        if (l == 0) tot = zz_ord64((double)c);
    } else {
        const zz_u64 ms = l < C ? mine[l * (W + 1) + W] : 0;
        const float m = l < C ? __uint_as_float((unsigned)ms) : -INFINITY, M = zz_wave_max(m);
        float part = l < C ? __uint_as_float((unsigned)(ms >> 32)) : 0.0f;
        if (m != M) part *= __builtin_amdgcn_exp2f((m - M) * ZZ_LOG2E);
        const double ls = log(zz_wave_sum((double)part));
        const zz_u64 b = zz_beam_best(mine, W + 1, C, W, P.cand[w]);
        const float L = zz_unord32((unsigned)(b >> 32));
        // the logit relative to its row's largest first: a row at the type's lowest value
        // keeps its bits; a row of minus infinities offers nothing better
        double t = (double)c + ((L == M ? 0.0 : (double)L - (double)M) - ls);
        if (t != t || M == -INFINITY) t = -(double)INFINITY;
        if (b && l < W) tot = zz_ord64(t);
        tok = (int)(0xffffffffu - (unsigned)b);
    }
    if (l < W) P.tot[w][l] = tot;
    __syncthreads();
    // A total's place is the number of better ones: its own list's before it, and in each other
    // list those not below it (equal totals go to the lower beam), found by halving. Lane l's
    // row of 16 lanes goes through every fourth list for the l % 16-th total.
    const int k = l & 15, part = l >> 4;
    const zz_u64 own = k < W ? P.tot[w][k] : 0;
    int at[ZZ_BEAM_MAXW / 4] = {};
#pragma unroll
    for (int s = 0; s < 5; s++) {
        const int step = s < 4 ? 8 >> s : 1;
#pragma unroll
        for (int j = 0; j < ZZ_BEAM_MAXW / 4; j++) {
            const int list = part + 4 * j;
            if (list < W && at[j] + step <= W && P.tot[list][at[j] + step - 1] >= own + (list > w)) at[j] += step;
        }
    }
    int rank = 0;
#pragma unroll
    for (int j = 0; j < ZZ_BEAM_MAXW / 4; j++) rank += part + 4 * j == w ? k : at[j];
    rank = zz_rows_sum(rank);
    if (l < W && own && rank < W) {
        const int o = blockIdx.x * W + rank;
        a.score_out[o] = (float)zz_unord64(own);
        a.parent[o] = w;
        a.token[o] = tok;
        if (a.done_out) a.done_out[o] = done || (a.eos >= 0 && tok == a.eos);
    }
}

// Dynamic LDS: each row's lists and sums, as the workspace holds them.
__global__ __launch_bounds__(1024) void zz_beam_merge_kernel(ZzBeamArgs a) {
    extern __shared__ __attribute__((aligned(16))) zz_u64 lists[];
    __shared__ ZzBeamPick P;
    const int w = zz_wave_id(), l = threadIdx.x & 63, row = blockIdx.x * a.W + w;
    // everything that is read, before anything waits: a finished beam's lists mean nothing, and
    // are not looked at
    const int words = a.chunks * (a.W + 1);
    zz_u64 *mine = lists + (size_t)w * words;
    const zz_u64 *from = a.ws + (size_t)row * words;
    const uint8_t done = a.done ? a.done[row] : 0;
    const float c = a.score[row];
#pragma unroll 8
    for (int i = l; i < words; i += 64) mine[i] = from[i];
    zz_wave_lds();
    zz_beam_finish(a, P, mine, a.chunks, done, c);
}

// A workgroup per sequence and a wave per beam, for rows that a wave's registers hold. One launch
// against two at 2048 f32 logits: 5.1 us against 6.0 (1 sequence of 4 beams), 6.9 against 7.1
// (1 of 8), 7.5 against 7.9 (32 of 8). Beyond 8 beams a workgroup's waves share their SIMDs and
// it loses: 8.5 against 7.9 (1 of 12), 10.8 against 8.9 (1 of 16).
#define ZZ_BEAM_SMALL 2048
template <typename T>
__global__ __launch_bounds__(512) void zz_beam_small_kernel(ZzBeamArgs a) {
    __shared__ ZzBeamPick P;
    __shared__ zz_u64 lists[8][ZZ_BEAM_MAXW + 1];
    const int w = zz_wave_id(), l = threadIdx.x & 63, W = a.W, row = blockIdx.x * W + w;
    const bool done = a.done && a.done[row];
    const float c = a.score[row];
    if (!done) {
        ZzBeamShare<T, ZZ_BEAM_SMALL * sizeof(T) / 1024> x((const T *)a.logits + row * a.ldl, a.V, l, 64);
        zz_u64 *best = lists[w], *cand = P.cand[w];
        const float lm = x.max(), m = zz_wave_max(lm), s = zz_wave_sum(x.sum(m));
        const int n = x.gather(zz_beam_line(lm, m, W, (float *)cand), cand);
        if (l < W) best[l] = 0;
        if (l == 0) best[W] = zz_beam_sum(m, s);
        zz_wave_lds();
        if (n <= 64) {
            const zz_u64 key = l < n ? cand[l] : 0;
            const int rank = zz_beam_place(key, n, cand);
            if (key && rank < W) best[rank] = key;
        } else {
            x.rounds(W, best);
        }
    }
    zz_wave_lds();
    zz_beam_finish(a, P, lists[w], 1, done, c);
}

// A thread owns 16 bytes of a row, at any alignment, in all W rows of a sequence: it reads what
// the W beams continue, then writes, so that moving in place needs no second buffer. Rows that
// stay where they are move nothing in place. The first workgroup moves the bytes behind the last
// whole piece as well.
// NT: the rows are stored past the caches, which their own dirty lines would fill (16 x 8 beams
// with 0.26 GB of states: the next step's pass over 134 MB of logits took 43 us instead of 32).
template <int WM, bool NT>
__global__ __launch_bounds__(256) void zz_beam_reorder_kernel(uint8_t *dst, const uint8_t *src, const int *parent, int W,
                                                              int64_t ostride, int64_t rstride, int64_t bytes) {
    const int n = blockIdx.y, tid = threadIdx.x;
    const int64_t base = blockIdx.z * ostride + (int64_t)n * W * rstride, pieces = bytes / 16;
    int par[WM];
#pragma unroll
    for (int w = 0; w < WM; w++) {
        const int p = w < W ? parent[n * W + w] : w;
        par[w] = p >= 0 && p < W ? p : w;
    }
    auto move = [&](auto piece, auto store, int64_t at) {
        typedef decltype(piece) G;
        G v[WM];
#pragma unroll
        for (int w = 0; w < WM; w++)
            if (w < W && (dst != src || par[w] != w)) v[w] = *(const G *)(src + at + par[w] * rstride);
#pragma unroll
        for (int w = 0; w < WM; w++)
            if (w < W && (dst != src || par[w] != w)) store(v[w], (G *)(dst + at + w * rstride));
    };
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < pieces; i += (int64_t)gridDim.x * 256)
        move(zz_u4any{}, [](zz_u4any v, zz_u4any *to) {
            if constexpr (NT) __builtin_nontemporal_store(v, to);
            else *to = v;
        }, base + i * 16);
    if (blockIdx.x == 0 && pieces * 16 + tid < bytes)
        move(uint8_t{}, [](uint8_t v, uint8_t *to) { *to = v; }, base + pieces * 16 + tid);
}

// ------------------------------------------------------------------ host side
int zz_lib_here(const char *who);                                             // zz_fp8.hip
int zz_ranges_meet(const void *a, int64_t n, const void *b, int64_t m);

// elements a thread holds: 32 (8192 a workgroup), or 8 where that leaves CUs without a workgroup
// and the lists to be joined stay few (4 rows of 32768 f32 logits 7.4 us a step against 7.6, of
// 128000 8.7 against 8.4)
static int beam_elems(int N, int W, int V) {
    return V <= 32 * 2048 && (int64_t)N * W * ((V + 8191) / 8192) < 256 ? 8 : 32;
}
static int beam_chunks(int N, int W, int V) {
    const int c = 256 * beam_elems(N, W, V);
    return (V + c - 1) / c;
}
static int beam_sizes_ok(int N, int W, int V) {
    return N >= 1 && W >= 1 && W <= ZZ_BEAM_MAXW && V >= 1 && V <= ZZ_BEAM_MAXV && (int64_t)N * W <= 65535;
}

extern "C" int64_t zz_beam_ws_bytes(int N, int W, int V) {
    if (!beam_sizes_ok(N, W, V)) return -1;
    return (int64_t)N * W * beam_chunks(N, W, V) * (W + 1) * 8;
}

extern "C" int zz_beam_step_dev(int dtype, const void *d_logits, int64_t ldl, int N, int W, int V,
                                const float *d_score, const uint8_t *d_done, int eos, int pad, float *d_score_out,
                                int *d_parent, int *d_token, uint8_t *d_done_out, void *d_ws, size_t ws_bytes,
                                void *stream) {
    const char *who = "zz_beam_step_dev";
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
    if (!beam_sizes_ok(N, W, V)) ZZ_FAIL("%s: 1 <= W <= %d, 1 <= V <= %d, 1 <= N * W <= 65535", who, ZZ_BEAM_MAXW, ZZ_BEAM_MAXV);
    if (!ldl) ldl = V;
    if (!d_logits || !d_score || !d_score_out || !d_parent || !d_token || !d_ws || ldl < V || ldl > (int64_t)1 << 40)
        ZZ_FAIL("%s: bad arguments", who);
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    if ((uintptr_t)d_logits % esz || (uintptr_t)d_score % 4 || (uintptr_t)d_score_out % 4 || (uintptr_t)d_parent % 4 ||
        (uintptr_t)d_token % 4 || (uintptr_t)d_ws % 8)
        ZZ_FAIL("%s: misaligned pointer", who);
    const int64_t need = zz_beam_ws_bytes(N, W, V);
    if (ws_bytes < (size_t)need) ZZ_FAIL("%s: %zu bytes of workspace, %lld needed", who, ws_bytes, (long long)need);
    const int64_t R = (int64_t)N * W;
    struct { const void *p; int64_t n; } in[] = {{d_logits, ((R - 1) * ldl + V) * esz}, {d_score, 4 * R}, {d_done, d_done ? R : 0}},
        out[] = {{d_score_out, 4 * R}, {d_parent, 4 * R}, {d_token, 4 * R}, {d_done_out, d_done_out ? R : 0}, {d_ws, need}};
    for (int i = 0; i < 5; i++) {
        for (int j = 0; j < 3; j++) {
            if ((i == 0 && j == 1 && out[i].p == in[j].p) || (i == 3 && j == 2 && out[i].p == in[j].p)) continue;
            if (out[i].n && in[j].n && zz_ranges_meet(out[i].p, out[i].n, in[j].p, in[j].n))
                ZZ_FAIL("%s: an output overlaps an input", who);
        }
        for (int j = 0; j < i; j++)
            if (out[i].n && out[j].n && zz_ranges_meet(out[i].p, out[i].n, out[j].p, out[j].n))
                ZZ_FAIL("%s: two outputs overlap", who);
    }
    if (!zz_lib_here(who)) return 0;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    if (V <= ZZ_BEAM_SMALL && W <= 8) {
        const ZzBeamArgs a{d_logits, ldl, N, W, V, 0, eos, pad, d_score, d_done, d_score_out, d_parent, d_token, d_done_out, nullptr};
        if (dtype == ZZ_F32) hipLaunchKernelGGL((zz_beam_small_kernel<float>), dim3(N), dim3(64 * W), 0, st, a);
        else hipLaunchKernelGGL((zz_beam_small_kernel<zz_bf16>), dim3(N), dim3(64 * W), 0, st, a);
        if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
        return 1;
    }
    const ZzBeamArgs a{d_logits, ldl, N, W, V, beam_chunks(N, W, V), eos, pad, d_score, d_done, d_score_out, d_parent,
                 d_token, d_done_out, (zz_u64 *)d_ws};
    const dim3 g(a.chunks, (unsigned)R), b(256);
    const bool few = beam_elems(N, W, V) == 8;
    if (dtype == ZZ_F32) {
        if (few) hipLaunchKernelGGL((zz_beam_part_kernel<float, 2>), g, b, 0, st, a);
        else hipLaunchKernelGGL((zz_beam_part_kernel<float, 8>), g, b, 0, st, a);
    } else {
        if (few) hipLaunchKernelGGL((zz_beam_part_kernel<zz_bf16, 1>), g, b, 0, st, a);
        else hipLaunchKernelGGL((zz_beam_part_kernel<zz_bf16, 4>), g, b, 0, st, a);
    }
    hipLaunchKernelGGL(zz_beam_merge_kernel, dim3(N), dim3(64 * W), (size_t)W * a.chunks * (W + 1) * 8, st, a);
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}

template <bool NT>
static void launch_reorder(uint8_t *dst, const uint8_t *src, const int *parent, int N, int W, int64_t outer,
                           int64_t ostride, int64_t rstride, int64_t bytes, hipStream_t st) {
    const int64_t gx = bytes < 256 * 16 ? 1 : bytes / 16 > 1024 * 256 ? 1024 : (bytes / 16 + 255) / 256;
    const auto k = W <= 4 ? zz_beam_reorder_kernel<4, NT> : W <= 8 ? zz_beam_reorder_kernel<8, NT> : zz_beam_reorder_kernel<16, NT>;
    for (int64_t o = 0; o < outer; o += 65535)                   // a grid's z dimension
        hipLaunchKernelGGL(k, dim3((unsigned)gx, N, (unsigned)(outer - o < 65535 ? outer - o : 65535)), dim3(256), 0, st,
                           dst + o * ostride, src + o * ostride, parent, W, ostride, rstride, bytes);
}

extern "C" int zz_beam_reorder_dev(void *d_dst, const void *d_src, const int *d_parent, int N, int W, int64_t outer,
                                   int64_t outer_stride, int64_t row_stride, int64_t row_bytes, void *stream) {
    const char *who = "zz_beam_reorder_dev";
    const int64_t far = (int64_t)1 << 40;
    if (!d_dst || !d_src || !d_parent || (uintptr_t)d_parent % 4 || N < 1 || W < 1 || W > ZZ_BEAM_MAXW ||
        (int64_t)N * W > 65535 || outer < 1 || outer > 1 << 20 || row_bytes < 1 || row_stride < row_bytes ||
        row_stride > far)
        ZZ_FAIL("%s: bad arguments (1 <= row_bytes <= row_stride, 1 <= W <= %d)", who, ZZ_BEAM_MAXW);
    const int64_t R = (int64_t)N * W;
    if (outer == 1) outer_stride = R * row_stride;               // there is no second plane
    if (outer_stride < R * row_stride || outer_stride > far) ZZ_FAIL("%s: planes overlap", who);
    const int64_t all = (outer - 1) * outer_stride + (R - 1) * row_stride + row_bytes;
    if (d_dst != d_src && zz_ranges_meet(d_dst, all, d_src, all)) ZZ_FAIL("%s: dst overlaps src", who);
    if (zz_ranges_meet(d_dst, all, d_parent, 4 * R)) ZZ_FAIL("%s: dst overlaps parent", who);
    if (!zz_lib_here(who)) return 0;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    uint8_t *d = (uint8_t *)d_dst;
    const uint8_t *s = (const uint8_t *)d_src;
    if (outer * R * row_bytes >= ZZ_NT_BYTES) launch_reorder<true>(d, s, d_parent, N, W, outer, outer_stride, row_stride, row_bytes, st);
    else launch_reorder<false>(d, s, d_parent, N, W, outer, outer_stride, row_stride, row_bytes, st);
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}
