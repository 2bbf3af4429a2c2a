// zz_experts.hip -- tokens to experts and back (include/zz_experts.h): the stable sort of the
// (token, slot) pairs by expert, the rows' copies, the weighted way back and its gradient.
//
// All of it moves rows and is bound by their bytes; the sort is bound by latency. A lane owns 8
// consecutive elements of a token's row (16 bytes of it, copied) and goes through the token's K
// pairs, so a token's row is read or written once and its K partners once each.
#include "zz_common.h"
#include "zz_kernels.h"
#include "zz_fp8_dev.h"
#include "../../include/zz_experts.h"

#define ZZ_FAIL(...)               \
    do {                           \
        zz_set_error(__VA_ARGS__); \
        return 0;                  \
    } while (0)

#define XP_FEW 1024                 // pairs that every workgroup looks through by itself
#define XP_ONE 8192                 // pairs that one workgroup sorts
#define XP_CHUNKS 256               // chunks of the others' sort

struct XpArgs {
    const int *eidx;
    int S, K, E, n;                 // n = S * K
    int *offs, *row, *pos;
    int chunk, chunks;              // pairs of a chunk, a multiple of 1024
    int *count;                     // [chunks][E]
    const uint8_t *x;               // rows as bytes, null: none
    uint8_t *xs;
    int64_t ldx, ldxs;              // bytes
    int bytes;                      // of a row
};

// A row's last unit, where its width leaves a rest, ends where the row ends and begins inside the
// unit before: vector loads all the same (element by element, a few lanes held their waves up: the
// way back of 8192 x 4 rows of 1087 bf16 took 45.8 us and takes 23.0, its
// bytes 20.9).
//
// `bytes` (a multiple of 2) of 16 bytes at any address
__device__ __forceinline__ zz_u4 xp_load(const uint8_t *p, int bytes) {
    if (bytes >= 16) return *(const zz_u4any *)p;
    zz_u4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 7; i++)
        if (2 * i + 2 <= bytes) v[i / 2] |= (unsigned)*(const uint16_t *)(p + 2 * i) << (16 * (i & 1));
    return v;
}
template <bool NT>
__device__ __forceinline__ void xp_store(uint8_t *p, zz_u4 v, int bytes) {
    if (bytes >= 16) {
        if constexpr (NT) __builtin_nontemporal_store((zz_u4any)v, (zz_u4any *)p);
        else *(zz_u4any *)p = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; i++)
        if (2 * i + 2 <= bytes) *(uint16_t *)(p + 2 * i) = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
}

// exclusive prefix sums of v[0 .. E) into offs[0 .. E] by one wave
template <typename PUT>
__device__ __forceinline__ void xp_offsets(const int *v, int E, PUT put) {
    constexpr int N = ZZ_EXPERTS_MAXE / 64;
    const int l = threadIdx.x & 63, per = (E + 63) / 64;
    int c[N], sum = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int e = l * per + i;
        c[i] = i < per && e < E ? v[e] : 0;
        sum += c[i];
    }
    const int upto = zz_wave_incl_scan_add(sum);
    int at = upto - sum;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int e = l * per + i;
        if (i < per && e < E) put(e, at);
        at += c[i];
    }
    if (l == 63) put(E, upto);
}

// Few pairs, one launch: a workgroup per token finds its pairs' positions by counting the pairs
// before them, one more the offsets.
__global__ __launch_bounds__(256) void zz_xp_few_kernel(XpArgs a) {
    __shared__ int hist[ZZ_EXPERTS_MAXE], part[4][ZZ_EXPERTS_MAXK], where[ZZ_EXPERTS_MAXK];
    const int tid = threadIdx.x, w = zz_wave_id(), l = tid & 63, s = blockIdx.x;
    int id[XP_FEW / 256];
#pragma unroll
    for (int i = 0; i < XP_FEW / 256; i++) id[i] = tid + 256 * i < a.n ? a.eidx[tid + 256 * i] : -1;
    if (s == a.S) {
        for (int e = tid; e < a.E; e += 256) hist[e] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < XP_FEW / 256; i++)
            if ((unsigned)id[i] < (unsigned)a.E) atomicAdd(&hist[id[i]], 1);
        __syncthreads();
        if (w == 0) xp_offsets(hist, a.E, [&](int e, int v) { a.offs[e] = v; });
        return;
    }
    const int ids = l < a.K ? a.eidx[s * a.K + l] : -1;   // the token's own
    int mine = 0;
    for (int k = 0; k < a.K; k++) {
        const int e = __builtin_amdgcn_readlane(ids, k), at = s * a.K + k;
        int c = 0;
#pragma unroll
        for (int i = 0; i < XP_FEW / 256; i++)
            c += __builtin_popcountll(__ballot((unsigned)id[i] < (unsigned)a.E && (id[i] < e || (id[i] == e && tid + 256 * i < at))));
        if (l == k) mine = c;
    }
    if (l < a.K) part[w][l] = mine;
    __syncthreads();
    if (tid < a.K) {
        const int p = (unsigned)ids < (unsigned)a.E ? part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid] : -1;
        a.pos[s * a.K + tid] = where[tid] = p;
        if (p >= 0) a.row[p] = s;
    }
    if (!a.x) return;
    __syncthreads();
    for (int u = 16 * tid; u < a.bytes; u += 4096) {
        const int b = max(min(u, a.bytes - 16), 0);
        const zz_u4 v = xp_load(a.x + s * a.ldx + b, a.bytes - b);
        for (int k = 0; k < a.K; k++)
            if (where[k] >= 0) xp_store<false>(a.xs + where[k] * a.ldxs + b, v, a.bytes - b);
    }
}

// how many pairs of each expert a chunk has
__global__ __launch_bounds__(1024) void zz_xp_count_kernel(XpArgs a) {
    __shared__ int hist[ZZ_EXPERTS_MAXE];
    const int tid = threadIdx.x, end = min(a.n, (int)(blockIdx.x + 1) * a.chunk);
    for (int e = tid; e < a.E; e += 1024) hist[e] = 0;
    __syncthreads();
    for (int i = blockIdx.x * a.chunk + tid; i < end; i += 1024) {
        const int e = a.eidx[i];
        if ((unsigned)e < (unsigned)a.E) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += 1024) a.count[blockIdx.x * a.E + e] = hist[e];
}

// The positions of a chunk's pairs. Each of 16 waves has a run of them: how many of an expert lie
// in the waves before is added up in LDS; within a wave's 64 pairs, the lanes with the same expert
// are found by a ballot for each bit of the id. Nothing depends on the order of atomics. A wave's
// pairs are requested 256 at a time; up to 256 it keeps for the second pass, more it requests again.
template <bool ONE>
__global__ __launch_bounds__(1024) void zz_xp_place_kernel(XpArgs a) {
    __shared__ int wcnt[16][ZZ_EXPERTS_MAXE], total[ZZ_EXPERTS_MAXE], pre[ZZ_EXPERTS_MAXE], base[ZZ_EXPERTS_MAXE + 1];
    const int tid = threadIdx.x, w = zz_wave_id(), l = tid & 63, E = a.E;
    const int per = a.chunk / 16, first = blockIdx.x * a.chunk + w * per, end = min(a.n, first + per);
    int id[4];
    auto take = [&](int from) {
#pragma unroll
        for (int i = 0; i < 4; i++) id[i] = from + 64 * i + l < end ? a.eidx[from + 64 * i + l] : -1;
    };
    take(first);
    for (int e = tid; e < E; e += 1024) total[e] = pre[e] = 0;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (tid < E) wcnt[i][tid] = 0;
    __syncthreads();
    for (int i0 = first; i0 < end; i0 += 256) {
        if (i0 != first) take(i0);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if ((unsigned)id[i] < (unsigned)E) atomicAdd(&wcnt[w][id[i]], 1);
    }
    if constexpr (!ONE) {                                 // the other chunks' pairs
        const int lanes = (E + 63) & ~63, groups = 1024 / lanes, e = tid % lanes, g = tid / lanes;
        if (e < E && g < groups) {
            int all = 0, before = 0;
#pragma unroll 4
            for (int c = g; c < a.chunks; c += groups) {
                const int v = a.count[c * E + e];
                all += v;
                before += c < (int)blockIdx.x ? v : 0;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&pre[e], before);
        }
    }
    __syncthreads();
    if (tid < E) {
        int t = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int v = wcnt[i][tid];
            wcnt[i][tid] = t;
            t += v;
        }
        if constexpr (ONE) total[tid] = t;
    }
    __syncthreads();
    if (w == 0)
        xp_offsets(total, E, [&](int e, int v) {
            base[e] = v;
            if (blockIdx.x == 0) a.offs[e] = v;
        });
    __syncthreads();
    const int bits = 32 - __builtin_clz(E);               // of an id, 0 .. E - 1
    if (per > 256) take(first);
    for (int i0 = first; i0 < end; i0 += 256) {
        if (i0 != first) take(i0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = i0 + 64 * i + l, e = id[i];
            const bool ok = (unsigned)e < (unsigned)E;
            unsigned long long same = __ballot(ok);
            for (int b = 0; b < bits; b++) {
                const unsigned long long m = __ballot(e >> b & 1);
                same &= e >> b & 1 ? m : ~m;
            }
            const int rank = __builtin_popcountll(same & ((1ull << l) - 1));
            int p = -1;
            if (ok) {
                const int before = wcnt[w][e];
                p = base[e] + (ONE ? 0 : pre[e]) + before + rank;
                asm volatile("" ::: "memory");            // all have read it
                if (rank == 0) wcnt[w][e] = before + __builtin_popcountll(same);
                a.row[p] = at / a.K;
            }
            asm volatile("" ::: "memory");
            if (at < end) a.pos[at] = p;
        }
    }
}

// the tokens' rows to their positions: 8192 x 8 of 2048 bf16 in 52 us, 5.8 TB/s
template <bool NT>
__global__ __launch_bounds__(256) void zz_xp_rows_kernel(XpArgs a) {
    const int units = (a.bytes + 15) / 16;
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    const int s = id / units, b = max(min(16 * (int)(id - s * units), a.bytes - 16), 0);
    if (s >= a.S) return;
    const zz_u4 v = xp_load(a.x + s * a.ldx + b, a.bytes - b);
#pragma unroll 8
    for (int k = 0; k < a.K; k++) {
        const int p = a.pos[s * a.K + k];
        if (p >= 0) xp_store<NT>(a.xs + p * a.ldxs + b, v, a.bytes - b);
    }
}

struct XpBack {
    const void *y, *res, *dout;
    const int *pos;
    const float *w;
    void *out, *dy;
    float *dw;
    int64_t ldy, ldr, ldo, ldg, lddy;   // elements
    int S, K, D, n;
};

// the position of pair i, -1 for none
__device__ __forceinline__ int xp_pos(const XpBack &a, int i) {
    const int p = a.pos[i];
    return (unsigned)p < (unsigned)a.n ? p : -1;
}

// 8 elements as they lie in memory, and as f32
template <typename T> struct XpRaw { zz_u4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ XpRaw<T> xp_raw(const T *p) {
    XpRaw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = *((const zz_u4any *)p + i);
    return r;
}
template <typename T>
__device__ __forceinline__ float xp_of(const XpRaw<T> &r, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[j >> 2][j & 3]);
    else return __uint_as_float(j & 1 ? r.w[0][j >> 1] & 0xffff0000u : r.w[0][j >> 1] << 16);
}
// a lane's unit of a row: 8 elements from e, of which the first `skip` are another lane's
struct XpUnit { int e, skip; };
__device__ __forceinline__ XpUnit xp_unit(int u, int D) {
    const int e = min(8 * u, D - 8);
    return {e, 8 * u - e};
}
template <bool NT, typename T>
__device__ __forceinline__ void xp_put(T *p, const float (&v)[8], int skip) {
    if (!skip) {
        zz_put8<NT>(p, v, 8);
        return;
    }
#pragma unroll
    for (int j = 1; j < 8; j++)
        if (j >= skip) zz_put(p + j, v[j]);
}

// Rows of fewer than 8 elements: a lane per element.
template <typename T>
__global__ __launch_bounds__(256) void zz_xp_back_narrow_kernel(XpBack a) {
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    const int s = id / a.D, e = id - s * a.D;
    if (s >= a.S) return;
    float v = a.res ? zz_f32_of(((const T *)a.res)[s * a.ldr + e]) : 0.0f;
    for (int k = 0; k < a.K; k++) {
        const int p = xp_pos(a, s * a.K + k);
        if (p >= 0) v = fmaf(a.w ? a.w[s * a.K + k] : 1.0f, zz_f32_of(((const T *)a.y)[p * a.ldy + e]), v);
    }
    zz_put((T *)a.out + s * a.ldo + e, v);
}

// 8 rows are on their way at once: 8192 x 16 of 64 bf16 7.1 us, one after the other 11.2. 8192 x 8
// rows of 2816 bf16 with a residual take 84 us, 5.5 TB/s.
template <typename T, bool NT>
__global__ __launch_bounds__(256) void zz_xp_back_kernel(XpBack a) {
    const int units = (a.D + 7) / 8;
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    const int s = id / units;
    if (s >= a.S) return;
    const XpUnit u = xp_unit(id - s * units, a.D);
    float v[8];
    if (a.res) {
        const XpRaw<T> r = xp_raw((const T *)a.res + s * a.ldr + u.e);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = xp_of(r, j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
    }
    for (int k0 = 0; k0 < a.K; k0 += 8) {
        int p[8];
        float w[8];
        XpRaw<T> r[8];
#pragma unroll
        for (int k = 0; k < 8; k++) p[k] = k0 + k < a.K ? xp_pos(a, s * a.K + k0 + k) : -1;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (p[k] >= 0) {
                r[k] = xp_raw((const T *)a.y + p[k] * a.ldy + u.e);
                w[k] = a.w ? a.w[s * a.K + k0 + k] : 1.0f;
            }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (p[k] >= 0)
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = fmaf(w[k], xp_of(r[k], j), v[j]);
    }
    xp_put<NT>((T *)a.out + s * a.ldo + u.e, v, u.skip);
}

// TPR lanes per token (a row of at most 8 TPR elements, or 256): they keep 8 elements of dout and go
// through the token's rows, 4 of them on their way at once; a row's sum is joined over the lanes.
// 4096 x 8 rows of 2816 bf16 take 76 us, 5.2 TB/s.
template <typename T, int TPR, bool NT>
__global__ __launch_bounds__(256) void zz_xp_grad_kernel(XpBack a) {
    __shared__ float part[4][ZZ_EXPERTS_MAXK];
    const int tid = threadIdx.x % TPR, units = (a.D + 7) / 8, l = threadIdx.x & 63;
    const int s = TPR == 256 ? blockIdx.x : blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool here = s < a.S;
    for (int k0 = 0; k0 < a.K; k0 += 4) {
        int p[4];
        float w[4], dot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            p[k] = here && k0 + k < a.K ? xp_pos(a, s * a.K + k0 + k) : -1;
            w[k] = p[k] >= 0 && a.w ? a.w[s * a.K + k0 + k] : 1.0f;
        }
        if (a.D >= 8) {
            for (int q = tid; q < units && here; q += TPR) {
                const XpUnit u = xp_unit(q, a.D);
                const XpRaw<T> g = xp_raw((const T *)a.dout + s * a.ldg + u.e);
                XpRaw<T> y[4];
                if (a.dw)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (p[k] >= 0) y[k] = xp_raw((const T *)a.y + p[k] * a.ldy + u.e);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (p[k] >= 0) {
                        float t[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            if (a.dw && j >= u.skip) dot[k] = fmaf(xp_of(g, j), xp_of(y[k], j), dot[k]);
                            t[j] = w[k] * xp_of(g, j);
                        }
                        xp_put<NT>((T *)a.dy + p[k] * a.lddy + u.e, t, u.skip);
                    }
            }
        } else if (tid < a.D && here) {
            const float g = zz_f32_of(((const T *)a.dout)[s * a.ldg + tid]);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (p[k] >= 0) {
                    if (a.dw) dot[k] = g * zz_f32_of(((const T *)a.y)[p[k] * a.ldy + tid]);
                    zz_put((T *)a.dy + p[k] * a.lddy + tid, w[k] * g);
                }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            dot[k] = zz_group_sum<TPR < 64 ? TPR : 64>(dot[k]);
            if (k0 + k >= a.K) continue;
            if constexpr (TPR == 256) {
                if (l == 0) part[zz_wave_id()][k0 + k] = dot[k];
            } else if (tid == 0 && here && a.dw) {
                a.dw[s * a.K + k0 + k] = dot[k];
            }
        }
    }
    if constexpr (TPR == 256) {
        __syncthreads();
        if (a.dw && tid < a.K) a.dw[s * a.K + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    }
}

template <typename T>
static void xp_launch_back(const XpBack &a, bool nt, hipStream_t st) {
    const int64_t t = (int64_t)a.S * (a.D < 8 ? a.D : (a.D + 7) / 8);
    const auto k = a.D < 8 ? zz_xp_back_narrow_kernel<T> : nt ? zz_xp_back_kernel<T, true> : zz_xp_back_kernel<T, false>;
    hipLaunchKernelGGL(k, dim3((unsigned)((t + 255) / 256)), dim3(256), 0, st, a);
}
template <typename T, int TPR>
static void xp_launch_grad(const XpBack &a, bool nt, hipStream_t st) {
    const auto k = nt ? zz_xp_grad_kernel<T, TPR, true> : zz_xp_grad_kernel<T, TPR, false>;
    hipLaunchKernelGGL(k, dim3((a.S + 256 / TPR - 1) / (256 / TPR)), dim3(256), 0, st, a);
}
// As few lanes a token as keep a narrow row's busy: with 256 for all, 8192 x 16 rows of 64 bf16 took
// 84 us and take 15, 4861 x 10 of 280 f32 51 and 30.
template <typename T>
static void xp_launch_grad(const XpBack &a, bool nt, hipStream_t st) {
    if (a.D <= 128) xp_launch_grad<T, 16>(a, nt, st);
    else if (a.D <= 1024) xp_launch_grad<T, 64>(a, nt, st);
    else xp_launch_grad<T, 256>(a, nt, st);
}

// ------------------------------------------------------------------ host side
int zz_lib_here(const char *who);                                             // zz_fp8.hip
int zz_ranges_meet(const void *a, int64_t n, const void *b, int64_t m);

static bool xp_sizes(int S, int K, int E) {
    return S >= 1 && S <= 1 << 20 && K >= 1 && K <= ZZ_EXPERTS_MAXK && E >= 1 && E <= ZZ_EXPERTS_MAXE;
}

// pairs of a chunk: at most XP_CHUNKS chunks of whole thousands
static int xp_chunk(int n) {
    if (n <= XP_ONE) return (n + 1023) / 1024 * 1024;
    const int c = ((n + XP_CHUNKS - 1) / XP_CHUNKS + 1023) / 1024 * 1024;
    return c < 4096 ? 4096 : c;
}

extern "C" int64_t zz_experts_ws_bytes(int S, int K, int E) {
    if (!xp_sizes(S, K, E)) return -1;
    const int n = S * K;
    return n <= XP_ONE ? 16 : (int64_t)((n + xp_chunk(n) - 1) / xp_chunk(n)) * E * 4;
}

// a range of memory; n = 0: none
struct XpRange { const void *p; int64_t n; };
static int64_t xp_span(int64_t ld, int64_t rows, int D, int esz) { return ((rows - 1) * ld + D) * esz; }

// whether one of `out` has a byte in common with one of `in` or with another of `out`
static bool xp_overlap(const XpRange *out, int no, const XpRange *in, int ni) {
    for (int i = 0; i < no; i++) {
        for (int j = 0; j < ni; j++)
            if (out[i].n && in[j].n && zz_ranges_meet(out[i].p, out[i].n, in[j].p, in[j].n)) return true;
        for (int j = 0; j < i; j++)
            if (out[i].n && out[j].n && zz_ranges_meet(out[i].p, out[i].n, out[j].p, out[j].n)) return true;
    }
    return false;
}

// a row distance: 0 becomes D; false where rows would overlap
static bool xp_ld(int64_t *ld, int D) {
    if (!*ld) *ld = D;
    return *ld >= D && *ld <= (int64_t)1 << 36;           // 2^24 rows' bytes stay under 2^62
}

extern "C" int zz_experts_dispatch_dev(const int *d_eidx, int S, int K, int E, int *d_offs, int *d_row, int *d_pos,
                                       int dtype, const void *d_x, int64_t ldx, int D, void *d_xs, int64_t ldxs,
                                       void *d_ws, size_t ws_bytes, void *stream) {
    const char *who = "zz_experts_dispatch_dev";
    if (!xp_sizes(S, K, E)) ZZ_FAIL("%s: S <= 2^20, K <= 16, E <= 512", who);
    if (!d_eidx || !d_offs || !d_row || !d_pos || !d_ws || (d_x && !d_xs)) ZZ_FAIL("%s: bad arguments", who);
    if (((uintptr_t)d_eidx | (uintptr_t)d_offs | (uintptr_t)d_row | (uintptr_t)d_pos | (uintptr_t)d_ws) % 4)
        ZZ_FAIL("%s: misaligned pointer", who);
    if (ws_bytes < (size_t)zz_experts_ws_bytes(S, K, E)) ZZ_FAIL("%s: the workspace is too small", who);
    const int n = S * K, esz = dtype == ZZ_F32 ? 4 : 2;
    if (d_x) {
        if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
        if (D < 1 || D > ZZ_MAXD) ZZ_FAIL("%s: 1 <= D <= %d", who, ZZ_MAXD);
        if (!xp_ld(&ldx, D) || !xp_ld(&ldxs, D)) ZZ_FAIL("%s: rows closer than their width", who);
        if (((uintptr_t)d_x | (uintptr_t)d_xs) % esz) ZZ_FAIL("%s: misaligned pointer", who);
    }
    const int64_t nxs = d_x ? xp_span(ldxs, n, D, esz) : 0;
    const XpRange out[] = {{d_offs, 4 * (int64_t)(E + 1)}, {d_row, 4 * (int64_t)n}, {d_pos, 4 * (int64_t)n},
                           {d_ws, zz_experts_ws_bytes(S, K, E)}, {d_xs, nxs}};
    const XpRange in[] = {{d_eidx, 4 * (int64_t)n}, {d_x, d_x ? xp_span(ldx, S, D, esz) : 0}};
    if (xp_overlap(out, 5, in, 2)) ZZ_FAIL("%s: an output overlaps another argument", who);
    if (!zz_lib_here(who)) return 0;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    XpArgs a;
    a.eidx = d_eidx; a.S = S; a.K = K; a.E = E; a.n = n; a.offs = d_offs; a.row = d_row; a.pos = d_pos;
    a.chunk = xp_chunk(n); a.chunks = (n + a.chunk - 1) / a.chunk; a.count = (int *)d_ws;
    a.x = (const uint8_t *)d_x; a.xs = (uint8_t *)d_xs; a.ldx = ldx * esz; a.ldxs = ldxs * esz; a.bytes = D * esz;
    if (n <= XP_FEW) {
        hipLaunchKernelGGL(zz_xp_few_kernel, dim3(S + 1), dim3(256), 0, st, a);
    } else {
        if (n <= XP_ONE) {
            hipLaunchKernelGGL(zz_xp_place_kernel<true>, dim3(1), dim3(1024), 0, st, a);
        } else {
            hipLaunchKernelGGL(zz_xp_count_kernel, dim3(a.chunks), dim3(1024), 0, st, a);
            hipLaunchKernelGGL(zz_xp_place_kernel<false>, dim3(a.chunks), dim3(1024), 0, st, a);
        }
        if (d_x) {
            const int64_t t = (int64_t)S * ((a.bytes + 15) / 16);
            const auto k = nxs >= ZZ_NT_BYTES ? zz_xp_rows_kernel<true> : zz_xp_rows_kernel<false>;
            hipLaunchKernelGGL(k, dim3((unsigned)((t + 255) / 256)), dim3(256), 0, st, a);
        }
    }
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}

extern "C" int zz_experts_back_dev(int dtype, const void *d_y, int64_t ldy, const int *d_pos, const float *d_w, int S,
                                   int K, int D, const void *d_res, int64_t ldr, void *d_out, int64_t ldo, void *stream) {
    const char *who = "zz_experts_back_dev";
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
    if (!xp_sizes(S, K, 1) || D < 1 || D > ZZ_MAXD) ZZ_FAIL("%s: S <= 2^20, K <= 16, D <= %d", who, ZZ_MAXD);
    if (!d_y || !d_pos || !d_out) ZZ_FAIL("%s: bad arguments", who);
    const int n = S * K, esz = dtype == ZZ_F32 ? 4 : 2;
    if (!xp_ld(&ldy, D) || !xp_ld(&ldo, D) || (d_res && !xp_ld(&ldr, D))) ZZ_FAIL("%s: rows closer than their width", who);
    if (((uintptr_t)d_y | (uintptr_t)d_res | (uintptr_t)d_out) % esz || ((uintptr_t)d_pos | (uintptr_t)d_w) % 4)
        ZZ_FAIL("%s: misaligned pointer", who);
    const bool own = d_res == d_out && ldr == ldo;
    const XpRange out = {d_out, xp_span(ldo, S, D, esz)};
    const XpRange in[] = {{d_y, xp_span(ldy, n, D, esz)}, {d_pos, 4 * (int64_t)n}, {d_w, d_w ? 4 * (int64_t)n : 0},
                          {d_res, d_res && !own ? xp_span(ldr, S, D, esz) : 0}};
    if (xp_overlap(&out, 1, in, 4)) ZZ_FAIL("%s: out overlaps another argument", who);
    if (!zz_lib_here(who)) return 0;
    XpBack a{};
    a.y = d_y; a.ldy = ldy; a.pos = d_pos; a.w = d_w; a.S = S; a.K = K; a.D = D; a.n = n; a.res = d_res; a.ldr = ldr;
    a.out = d_out; a.ldo = ldo;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    dtype == ZZ_F32 ? xp_launch_back<float>(a, out.n >= ZZ_NT_BYTES, st) : xp_launch_back<zz_bf16>(a, out.n >= ZZ_NT_BYTES, st);
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}

extern "C" int zz_experts_back_grad_dev(int dtype, const void *d_dout, int64_t ldg, const void *d_y, int64_t ldy,
                                        const int *d_pos, const float *d_w, int S, int K, int D, void *d_dy, int64_t lddy,
                                        float *d_dw, void *stream) {
    const char *who = "zz_experts_back_grad_dev";
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
    if (!xp_sizes(S, K, 1) || D < 1 || D > ZZ_MAXD) ZZ_FAIL("%s: S <= 2^20, K <= 16, D <= %d", who, ZZ_MAXD);
    if (!d_dout || !d_pos || !d_dy || (d_dw && !d_y)) ZZ_FAIL("%s: bad arguments", who);
    const int n = S * K, esz = dtype == ZZ_F32 ? 4 : 2;
    if (!xp_ld(&ldg, D) || !xp_ld(&lddy, D) || (d_dw && !xp_ld(&ldy, D))) ZZ_FAIL("%s: rows closer than their width", who);
    if (((uintptr_t)d_dout | (uintptr_t)d_dy | (d_dw ? (uintptr_t)d_y : 0)) % esz ||
        ((uintptr_t)d_pos | (uintptr_t)d_w | (uintptr_t)d_dw) % 4)
        ZZ_FAIL("%s: misaligned pointer", who);
    const bool own = d_dy == d_y && lddy == ldy;
    const XpRange out[] = {{d_dy, xp_span(lddy, n, D, esz)}, {d_dw, d_dw ? 4 * (int64_t)n : 0}};
    const XpRange in[] = {{d_dout, xp_span(ldg, S, D, esz)}, {d_pos, 4 * (int64_t)n}, {d_w, d_w ? 4 * (int64_t)n : 0},
                          {d_y, d_dw && !own ? xp_span(ldy, n, D, esz) : 0}};
    if (xp_overlap(out, 2, in, 4)) ZZ_FAIL("%s: an output overlaps another argument", who);
    if (!zz_lib_here(who)) return 0;
    XpBack a{};
    a.dout = d_dout; a.ldg = ldg; a.y = d_y; a.ldy = ldy; a.pos = d_pos; a.w = d_w; a.S = S; a.K = K; a.D = D; a.n = n;
    a.dy = d_dy; a.lddy = lddy; a.dw = d_dw;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    const bool nt = out[0].n >= ZZ_NT_BYTES;
    dtype == ZZ_F32 ? xp_launch_grad<float>(a, nt, st) : xp_launch_grad<zz_bf16>(a, nt, st);
    if (hipGetLastError() != hipSuccess) ZZ_FAIL("%s: launch failed", who);
    return 1;
}
