// zz_fp8_ep.h -- the fp8 product with bias, activation, gate and residual in its epilogue, for
// one matrix or a table of experts (include/zz_fp8.h). Instantiated by zz_fp8_ep.hip (G = 1) and
// zz_fp8_gated.hip (G = 2).
//
//   v = sum_b xs[b][r] ws[..][b] sum_{k in b} xq[r][k] wq[o][k] + bias[o],  r = row[p]
//   y[p][o] = act(v) + res[p][o], or act(min(v_gate, c)) * clip(v_up, -c, c) + res[p][o]
// The sums are those of zz_fp8_mma.h. An expert's rows lie side by side in y: a workgroup's tile
// belongs to one expert, and its place is found from the experts' offsets, which only the device
// knows, by a scan over them in registers: no list, no second launch.
#pragma once
#include "zz_fp8_mma.h"

// Row tile t of the experts' tiles of TS rows, or with OT columns of tiles the t-th tile of all:
// its expert, that expert's first row and rows, and the row tiles before the expert's. Each wave
// counts them for itself, 64 experts at a time. False: there is no such tile.
struct ZzF8Found { int e, first, rows, before; };
template <int TS, bool XCD>
__device__ __forceinline__ bool zz_f8_find(const ZzF8Ep &a, int OT, int &t, ZzF8Found &f) {
    constexpr int NC = ZZ_F8_MAXE / 64;
    const int l = threadIdx.x & 63;
    int lo[NC], n[NC], upto[NC], total = 0;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        lo[c] = n[c] = 0;
        if (64 * c < a.E) {
            lo[c] = a.offs[min(64 * c + l, a.E)];
            n[c] = a.offs[min(64 * c + l + 1, a.E)];
        }
    }
#pragma unroll
    for (int c = 0; c < NC; c++) {
        lo[c] = min(max(lo[c], 0), a.P);                  // whatever they hold, rows of y are inside
        n[c] = max(min(max(n[c], 0), a.P) - lo[c], 0);
        upto[c] = total;
        if (64 * c < a.E) {
            upto[c] += zz_wave_incl_scan_add((n[c] + TS - 1) / TS);
            total = __builtin_amdgcn_readlane(upto[c], 63);
        }
    }
    int row = t;
    if constexpr (XCD) {
        const int per = (total * OT + 7) / 8;
        const int id = t % 8 * per + t / 8;
        if (t / 8 >= per || id >= total * OT) return false;
        t = id;
        row = id / OT;
    } else if (t >= total) {
        return false;
    }
    bool open = true;
#pragma unroll
    for (int c = 0; c < NC; c++)
        if (open && row < __builtin_amdgcn_readlane(upto[c], 63)) {
            const int at = (int)__builtin_ctzll(__ballot(upto[c] > row));
            f.e = 64 * c + at;
            f.first = __builtin_amdgcn_readlane(lo[c], at);
            f.rows = __builtin_amdgcn_readlane(n[c], at);
            f.before = __builtin_amdgcn_readlane(upto[c], at) - (f.rows + TS - 1) / TS;
            open = false;
        }
    return true;
}

// the arguments of that expert's product alone
template <int G, typename T>
__device__ __forceinline__ void zz_f8_expert(ZzF8Ep &a, const ZzF8Found &f) {
    a.m.w += f.e * a.we;
    a.m.ws += (int64_t)f.e * a.wse;
    if (a.bias) a.bias += (int64_t)f.e * a.m.O * G;
    a.S = f.rows;
    a.y = (T *)a.y + f.first * a.ldy;
    if (a.res) a.res = (const T *)a.res + f.first * a.ldr;
    if (a.row) {
        a.row += f.first;
    } else {
        a.q += (int64_t)f.first * a.nb * ZZ_F8B;
        a.s += f.first;
    }
}

template <typename T, int G, int RG, int RS, int NW, bool PF, bool NT>
__global__ __launch_bounds__(64 * NW) void zz_fp8_few_ep_kernel(ZzF8Ep a) {
    extern __shared__ __attribute__((aligned(16))) float part[];
    constexpr int OC = RG * zz_f8_gw<G>;
    const int OT = (a.m.O + OC - 1) / OC;
    int st = blockIdx.x / OT;
    if (a.offs) {
        ZzF8Found f;
        if (!zz_f8_find<32 * RS, false>(a, 1, st, f)) return;
        zz_f8_expert<G, T>(a, f);
        st -= f.before;
    }
    zz_fp8_few<T, G, RG, RS, NW, PF, NT>(a, part, blockIdx.x % OT * RG, st * 32 * RS);
}

// A workgroup's tile of 32 TG packed rows x TS rows: its column and row tile, the arguments made
// its expert's. Tiles go XCD by XCD in the order of the experts, so that an expert's codes are read
// into one XCD's L2.
template <int G, typename T, int TG, int TS>
__device__ __forceinline__ bool zz_f8_place(ZzF8Ep &a, int *ot, int *st) {
    constexpr int OC = TG * zz_f8_gw<G>;
    const int OT = (a.m.O + OC - 1) / OC;
    int id = blockIdx.x;
    if (a.offs) {
        ZzF8Found f;
        if (!zz_f8_find<TS, true>(a, OT, id, f)) return false;
        zz_f8_expert<G, T>(a, f);
        id -= f.before * OT;
    } else {
        id = id % 8 * (gridDim.x / 8) + id / 8;
        if (id >= (a.S + TS - 1) / TS * OT) return false;
    }
    zz_fp8_at(id, OT, (a.S + TS - 1) / TS, ot, st);
    return true;
}

template <typename T, int G, int RO, int RS, int WO, int WS, int KS, int NS, bool NT>
__global__ __launch_bounds__(64 * WO * WS * KS, 2) void zz_fp8_tiles_ep_kernel(ZzF8Ep a) {
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    int ot, st;
    if (!zz_f8_place<G, T, C::O / 32, C::S>(a, &ot, &st)) return;
    zz_fp8_tile<T, G, RO, RS, WO, WS, KS, NS, NT>(a, lds, ot * C::O / 32, st * C::S);
}

template <typename T, int G, int RG, int RS, int NW, bool PF, bool NT>
static bool launch_few_ep(const ZzF8EpCall &c, const ZzF8Ep &a, hipStream_t st) {
    constexpr int OC = RG * zz_f8_gw<G>;
    const int64_t n = zz_f8_ep_tiles(c.P, c.E, c.offs, 32 * RS) * ((a.m.O + OC - 1) / OC);
    if (!zz_f8_fits(n, 64 * NW)) return false;
    hipLaunchKernelGGL((zz_fp8_few_ep_kernel<T, G, RG, RS, NW, PF, NT>), dim3((unsigned)n), dim3(64 * NW), NW * RG * RS * 4096, st, a);
    return true;
}

template <typename C, int G>
static bool launch_tiles_ep(const ZzF8EpCall &c, const ZzF8Ep &a, void (*kernel)(ZzF8Ep), hipStream_t st) {
    constexpr int OC = C::O / 32 * zz_f8_gw<G>;
    const int64_t n = (zz_f8_ep_tiles(c.P, c.E, c.offs, C::S) * ((a.m.O + OC - 1) / OC) + 7) / 8 * 8;
    if (!zz_f8_fits(n, C::NT)) return false;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(C::NT), C::LDS, st, a);
    return true;
}

template <typename T, int G, int RO, int RS, int WO, int WS, int KS, int NS, bool CANNT>
static bool launch_async_ep(const ZzF8EpCall &c, const ZzF8Ep &a, hipStream_t st) {
    typedef ZzF8Async<RO, RS, WO, WS, KS, NS> C;
    return launch_tiles_ep<C, G>(c, a, CANNT && a.nt ? zz_fp8_tiles_ep_kernel<T, G, RO, RS, WO, WS, KS, NS, CANNT>
                                                     : zz_fp8_tiles_ep_kernel<T, G, RO, RS, WO, WS, KS, NS, false>, st);
}

#include "zz_fp8_wide.h"

template <typename T, int G>
static bool launch_ep(const ZzF8EpCall &c, hipStream_t st) {
    ZzF8Ep a;
    a.m = c.m; a.q = c.q; a.s = c.s; a.S = c.P; a.nb = zz_f8_nb(c.m.I); a.y = c.y; a.ldy = c.ldy;
    a.R = c.R; a.row = c.row; a.bias = c.bias; a.res = c.res; a.ldr = c.ldr; a.act = c.act; a.clamp = c.clamp;
    a.offs = c.offs; a.E = c.E; a.P = c.P; a.we = c.we; a.wse = c.wse; a.wsu = c.wsu;
    // large results past the caches where tiles write whole lines, as zz_fp8_mma.hip's
    a.nt = c.P * a.ldy * (int64_t)sizeof(T) >= ZZ_NT_BYTES && (uintptr_t)a.y % 64 == 0 && a.ldy * sizeof(T) % 64 == 0;
    const int v = zz_f8_ep_kernel(G * c.m.O, c.m.I, c.P, c.E, c.offs != nullptr, sizeof(T) == 2 && c.eight);
    bool ok = false;
    if (v == 0) ok = launch_few_ep<T, G, 1, 1, 16, false, false>(c, a, st);
    else if (v == 1) ok = launch_few_ep<T, G, 1, 1, 4, true, false>(c, a, st);
    else if (v == 2) ok = launch_few_ep<T, G, 2, 1, 8, false, false>(c, a, st);
    else if (v == 3) ok = launch_async_ep<T, G, 1, 1, 2, 1, 2, 2, false>(c, a, st);
    else if (v == 4) ok = launch_async_ep<T, G, 1, 2, 2, 1, 4, 2, false>(c, a, st);
    else if (v == 5) ok = launch_async_ep<T, G, 1, 2, 2, 1, 2, 2, false>(c, a, st);
    else if (v == 14) ok = launch_few_ep<T, G, 1, 1, 4, true, true>(c, a, st);
    else if (v == 15) ok = launch_few_ep<T, G, 1, 1, 8, true, true>(c, a, st);
    else if (v == 16) ok = launch_few_ep<T, G, 2, 1, 4, true, true>(c, a, st);
    if (ok) return true;
    // the largest tiles also where smaller ones are more than a launch holds
    if constexpr (sizeof(T) == 2) {
        if (v == 11 && launch_wide<G, 2, 2, 2>(c, a, st)) return true;
        if (v == 12 && launch_wide<G, 2, 4, 3>(c, a, st)) return true;
        if (v >= 11 && v <= 13) return launch_wide<G, 4, 4, 2>(c, a, st);
    }
    if (v == 6 && launch_async_ep<T, G, 1, 1, 2, 2, 1, 3, false>(c, a, st)) return true;
    if (v == 7 && launch_async_ep<T, G, 1, 2, 2, 2, 1, 2, true>(c, a, st)) return true;
    return launch_async_ep<T, G, 2, 2, 2, 2, 1, 2, true>(c, a, st);
}
