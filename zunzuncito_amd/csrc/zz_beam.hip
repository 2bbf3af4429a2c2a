// zz_beam.hip -- beam search's step (include/zz_beam.h).
//
//   total(w, t) = score[w] + ((L[w][t] - m[w]) - log(sum_t exp(L[w][t] - m[w]))), m the maximum
// Within a row totals go by the logit, so a row's W best are found on the logits alone, as
// 64-bit keys (order-preserving bits of the logit, then the lower token), and the sum of
// exponentials belongs to the same pass over the data. Two launches:
//   zz_beam_part_kernel   a workgroup per (row, chunk of the vocabulary): the chunk's W
//                         largest keys in order, its maximum and sum of exponentials
//   zz_beam_merge_kernel  a workgroup per sequence: a wave per beam joins the chunks' lists
//                         and sums (in double), then one wave picks the W best totals
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

// the wave's largest key: the upper words first, the lower ones only where several lanes share
// the upper word (equal logits)
__device__ __forceinline__ zz_u64 zz_wave_max64(zz_u64 v) {
    const unsigned hi = (unsigned)(v >> 32), lo = (unsigned)v;
    auto mx = [](unsigned a, unsigned b) { return a > b ? a : b; };
    const unsigned H = zz_group_reduce<64>(hi, mx);
    const zz_u64 at = __ballot(hi == H);
    unsigned L;
    if (__popcll(at) == 1) L = (unsigned)__builtin_amdgcn_readlane((int)lo, __ffsll((long long)at) - 1);
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

// NV pieces of 16 bytes a thread, piece i * 256 + tid of the chunk counted from the row's first
// token: the sum's order does not depend on where the row lies, so equal rows have equal
// totals. A row of an odd vocabulary begins at any multiple of its element; the loads need no
// more. The pieces across the row's end go element by element.
template <typename T, int NV>
__global__ __launch_bounds__(256) void zz_beam_part_kernel(ZzBeamArgs a) {
    constexpr int VE = 16 / sizeof(T), NE = NV * VE;
    __shared__ zz_u64 cand[4][64];
    __shared__ zz_u64 best[4][ZZ_BEAM_MAXW];
    __shared__ float wm[4], wsum[4];
    const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x, l = tid & 63, w = tid >> 6, W = a.W, V = a.V;
    if (a.done && a.done[row]) return;
    const T *L = (const T *)a.logits + row * a.ldl;
    float v[NE];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = (ch * NV * 256 + i * 256 + tid) * VE;
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
    // the token of element k, or -1 where it lies outside the row
    auto tok = [&](int k) {
        const int t = (ch * NV * 256 + (k / VE) * 256 + tid) * VE + k % VE;
        return t < V ? t : -1;
    };
    float lm = -INFINITY;
#pragma unroll
    for (int k = 0; k < NE; k++) {
        v[k] = fmaxf(v[k], -INFINITY);                   // a NaN counts as minus infinity
        lm = fmaxf(lm, v[k]);
    }
    const float m = zz_wave_max(lm);
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
    s = zz_wave_sum(s);
    // The W-th largest of the lanes' maxima: at least W logits reach it, and the W best do. What
    // reaches it is a few more than W, unless many are equal.
    float left = lm, line = m;
    for (int k = 1; k < W; k++) {
        const zz_u64 at = __ballot(left == line);
        if (l == __ffsll((long long)at) - 1) left = -INFINITY;
        line = zz_wave_max(left);
    }
    if (l < W) best[w][l] = 0;
    cand[w][l] = 0;
    int total = line == -INFINITY ? 65 : 0;              // padding would be among them
    if (total == 0) {
#pragma unroll
        for (int k = 0; k < NE; k++) {
            const zz_u64 at = __ballot(v[k] >= line);
            if (at) {
                const int o = total + __builtin_amdgcn_mbcnt_hi((unsigned)(at >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)at, 0));
                if (v[k] >= line && o < 64) cand[w][o] = zz_beam_key(v[k], tok(k));
                total += __popcll(at);
            }
        }
    }
    if (total <= 64) {
        // a candidate a lane: its place is the number of better ones
        const zz_u64 key = cand[w][l];
        int rank = 0;
        for (int j = 0; j < total; j += 8)
#pragma unroll
            for (int i = 0; i < 8; i++) rank += cand[w][j + i] > key;
        if (l < total && rank < W) best[w][rank] = key;
    } else {
        // W rounds of the wave's largest remaining key
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
            if (l == 0) best[w][k] = prev;
        }
    }
    if (l == 0) { wm[w] = m; wsum[w] = s; }
    __syncthreads();
    if (w != 0) return;
    // the four waves' lists, a key a lane: its place among all is the number of better ones
    const zz_u64 key = l < 4 * W ? best[l / W][l % W] : 0;
    cand[0][l] = key;
    int rank = 0;
    for (int j = 0; j < 4 * W; j += 4)
#pragma unroll
        for (int i = 0; i < 4; i++) rank += cand[0][j + i] > key || (cand[0][j + i] == key && j + i < l);
    zz_u64 *out = a.ws + ((size_t)row * a.chunks + ch) * (W + 1);
    if (l < 4 * W && rank < W) out[rank] = key;
    if (l == 0) {
        const float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
        float t = 0.0f;
        for (int q = 0; q < 4; q++) t += wm[q] == M ? wsum[q] : wsum[q] * __builtin_amdgcn_exp2f((wm[q] - M) * ZZ_LOG2E);
        out[W] = ((zz_u64)__float_as_uint(t) << 32) | __float_as_uint(M);
    }
}

// Dynamic LDS: each row's lists and sums, as the workspace holds them.
__global__ __launch_bounds__(1024) void zz_beam_merge_kernel(ZzBeamArgs a) {
    extern __shared__ __attribute__((aligned(16))) zz_u64 lists[];
    __shared__ zz_u64 tot[ZZ_BEAM_MAXW][ZZ_BEAM_MAXW];      // ordered totals, 0: no candidate
    __shared__ int tk[ZZ_BEAM_MAXW][ZZ_BEAM_MAXW];
    __shared__ uint8_t fin[ZZ_BEAM_MAXW];
    const int n = blockIdx.x, w = zz_wave_id(), l = threadIdx.x & 63, W = a.W, row = n * W + w, C = a.chunks;
    // everything that is read, before anything waits: a finished beam's lists mean nothing, and
    // are not looked at
    const int words = C * (W + 1);
    zz_u64 *mine = lists + (size_t)w * words;
    const zz_u64 *from = a.ws + (size_t)row * words;
    const uint8_t flag = a.done ? a.done[row] : 0;
    float c = a.score[row];
#pragma unroll 8
    for (int i = l; i < words; i += 64) mine[i] = from[i];
    const bool done = flag;
    if (c != c) c = -INFINITY;
    if (done) {
        if (l < W) {
            tot[w][l] = l == 0 ? zz_ord64((double)c) : 0;
            tk[w][l] = a.pad;
        }
    } else {
        const zz_u64 *p = mine + l * (W + 1);
        const zz_u64 ms = l < C ? p[W] : 0;
        const float m = l < C ? __uint_as_float((unsigned)ms) : -INFINITY, M = zz_wave_max(m);
        float part = l < C ? __uint_as_float((unsigned)(ms >> 32)) : 0.0f;
        if (m != M) part *= __builtin_amdgcn_exp2f((m - M) * ZZ_LOG2E);
        const double s = zz_wave_sum((double)part);
        const double ls = log(s);
        // the chunks' sorted lists, one a lane: W times the largest head
        int at = 0;
        zz_u64 head = l < C ? p[0] : 0;
        for (int k = 0; k < W; k++) {
            const zz_u64 b = zz_wave_max64(head);
            if (l == k) {
                const float L = zz_unord32((unsigned)(b >> 32));
                // the logit relative to its row's largest first: a row at the type's lowest value
                // keeps its bits; a row of minus infinities offers nothing better
                double t = (double)c + ((L == M ? 0.0 : (double)L - (double)M) - ls);
                if (t != t || M == -INFINITY) t = -(double)INFINITY;
                tot[w][k] = b ? zz_ord64(t) : 0;
                tk[w][k] = (int)(0xffffffffu - (unsigned)b);
            }
            if (head == b && b) {
                at++;
                head = at < W ? p[at] : 0;
            }
        }
    }
    if (l == 0) fin[w] = done;
    __syncthreads();
    if (w != 0) return;
    // the beams' lists, one a lane; equal totals go to the lower beam
    int at = 0;
    zz_u64 head = l < W ? tot[l][0] : 0;
    for (int k = 0; k < W; k++) {
        const zz_u64 b = zz_wave_max64(head);
        const int who = __ffsll((long long)__ballot(head == b && l < W)) - 1;
        if (l == who) {
            const int o = n * W + k, t = tk[l][at];
            a.score_out[o] = (float)zz_unord64(b);
            a.parent[o] = l;
            a.token[o] = t;
            if (a.done_out) a.done_out[o] = fin[l] || (a.eos >= 0 && t == a.eos);
            at++;
            head = at < W ? tot[l][at] : 0;
        }
    }
}

// A thread owns one piece G of a row's bytes in all W rows of a sequence: it reads what
// the W beams continue, then writes, so that moving in place needs no second buffer. Rows
// that stay where they are move nothing in place.
// NT: the rows are stored past the caches, which their own dirty lines would fill (16 x 8 beams
// with 0.26 GB of states: the next step's pass over 134 MB of logits took 43 us instead of 32).
template <typename G, int WM, bool NT>
__global__ __launch_bounds__(256) void zz_beam_reorder_kernel(uint8_t *dst, const uint8_t *src, const int *parent, int W,
                                                              int64_t ostride, int64_t rstride, int64_t first,
                                                              int64_t pieces) {
    const int n = blockIdx.y, tid = threadIdx.x;
    const int64_t o = blockIdx.z;
    const int64_t base = o * ostride + (int64_t)n * W * rstride + first;
    int par[WM];
#pragma unroll
    for (int w = 0; w < WM; w++) {
        const int p = w < W ? parent[n * W + w] : w;
        par[w] = p >= 0 && p < W ? p : w;
    }
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t at = base + i * (int64_t)sizeof(G);
        G v[WM];
#pragma unroll
        for (int w = 0; w < WM; w++)
            if (w < W && (dst != src || par[w] != w)) v[w] = *(const G *)(src + at + par[w] * rstride);
#pragma unroll
        for (int w = 0; w < WM; w++)
            if (w < W && (dst != src || par[w] != w)) {
                G *to = (G *)(dst + at + w * rstride);
                if constexpr (NT) __builtin_nontemporal_store(v[w], to);
                else *to = v[w];
            }
    }
}

// ------------------------------------------------------------------ host side
int zz_lib_here(const char *who);                                             // zz_fp8.hip
int zz_ranges_meet(const void *a, int64_t n, const void *b, int64_t m);

// elements a thread holds: 32 (8192 a workgroup), or 8 where that leaves too few workgroups
static int beam_elems(int N, int W, int V) {
    return V <= 64 * 2048 && (int64_t)N * W * ((V + 8191) / 8192) < 512 ? 8 : 32;
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
    ZzBeamArgs a{d_logits, ldl, N, W, V, beam_chunks(N, W, V), eos, pad, d_score, d_done, d_score_out, d_parent,
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

template <typename G, bool NT>
static void launch_reorder(uint8_t *dst, const uint8_t *src, const int *parent, int N, int W, int64_t outer,
                           int64_t ostride, int64_t rstride, int64_t first, int64_t pieces, hipStream_t st) {
    int64_t gx = (pieces + 255) / 256;
    if (gx > 1024) gx = 1024;
    const auto k = W <= 4 ? zz_beam_reorder_kernel<G, 4, NT>
                          : W <= 8 ? zz_beam_reorder_kernel<G, 8, NT> : zz_beam_reorder_kernel<G, 16, NT>;
    for (int64_t o = 0; o < outer; o += 65535)                   // a grid's z dimension
        hipLaunchKernelGGL(k, dim3((unsigned)gx, N, (unsigned)(outer - o < 65535 ? outer - o : 65535)), dim3(256), 0, st,
                           dst + o * ostride, src + o * ostride, parent, W, ostride, rstride, first, pieces);
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
    // pieces as wide as every row's alignment allows, then the bytes behind the last whole one
    const uintptr_t al = (uintptr_t)d | (uintptr_t)s | (uintptr_t)row_stride | (outer > 1 ? (uintptr_t)outer_stride : 0);
    const int64_t gsz = al % 16 == 0 ? 16 : al % 4 == 0 ? 4 : 1, body = row_bytes / gsz, tail = row_bytes - body * gsz;
    auto move = [&](auto launch, int64_t first, int64_t n) {
        if (n) launch(d, s, d_parent, N, W, outer, outer_stride, row_stride, first, n, st);
    };
    if (gsz == 16 && outer * R * row_bytes >= ZZ_NT_BYTES) move(launch_reorder<zz_u4, true>, 0, body);
    else if (gsz == 16) move(launch_reorder<zz_u4, false>, 0, body);
    else if (gsz == 4) move(launch_reorder<unsigned, false>, 0, body);
    else move(launch_reorder<uint8_t, false>, 0, body);
    move(launch_reorder<uint8_t, false>, body * gsz, tail);
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}
