// zz_fp8.hip -- host side of include/zz_fp8.h: the checks of arguments, the resident
// matrices and the host form.
#include "zz_common.h"
#include "zz_kernels.h"
#include "zz_fp8_dev.h"
#include "../../include/zz_fp8.h"

#include <math.h>
#include <new>
#include <vector>

#define ZZ_FAIL(...)               \
    do {                           \
        zz_set_error(__VA_ARGS__); \
        return 0;                  \
    } while (0)

#define ZZ_F8_MAXS (1 << 20)
#define ZZ_F8_MAXNORM 8192
#define ZZ_F8_MAXP (1 << 24)

// the library is up and its device is the current one; the last check of a call, so that
// what is wrong with its arguments is named without a device too
int zz_lib_here(const char *who) {
    int dev = -1;
    if (!zz_lib_ready() || hipGetDevice(&dev) != hipSuccess || dev != 0)
        ZZ_FAIL("%s: gpu_init first, and its device has to be the current one", who);
    return 1;
}

// whether [a, a + n) and [b, b + m) have a byte in common
int zz_ranges_meet(const void *a, int64_t n, const void *b, int64_t m) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uint64_t)m && y < x + (uint64_t)n;
}

extern "C" int64_t zz_fp8_row_bytes(int64_t D) {
    return D < 1 ? -1 : (D + ZZ_F8B - 1) / ZZ_F8B * ZZ_F8B;
}

static int rows_common(const char *who, int dtype, const void *x, int64_t *ldx, int S, int most, int D, const uint8_t *q,
                       const float *s) {
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
    if (!x || !q || !s || S < 1 || S > most || D < 1) ZZ_FAIL("%s: bad arguments (1 <= S <= %d)", who, most);
    if (!*ldx) *ldx = D;
    // S rows' bytes stay under 2^62
    if (*ldx < D || *ldx > (int64_t)1 << (S > ZZ_F8_MAXS ? 36 : 40)) ZZ_FAIL("%s: rows closer than their width", who);
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    if ((uintptr_t)x % esz || (uintptr_t)q % 16 || (uintptr_t)s % 4) ZZ_FAIL("%s: misaligned pointer", who);
    return 1;
}

static int64_t span(int64_t ld, int S, int D, int esz) { return ((S - 1) * ld + D) * esz; }

extern "C" int zz_add_norm_fp8_dev(int dtype, const void *d_x, int64_t ldx, const void *d_res, int64_t ldr,
                                   void *d_sum, int64_t lds, const float *d_w, float eps, int S, int D,
                                   uint8_t *d_q, float *d_s, void *stream) {
    const char *who = "zz_add_norm_fp8_dev";
    if (!rows_common(who, dtype, d_x, &ldx, S, ZZ_F8_MAXS, D, d_q, d_s)) return 0;
    if (D > ZZ_F8_MAXNORM) ZZ_FAIL("%s: D <= %d", who, ZZ_F8_MAXNORM);
    if (!(eps >= 0.0f) || isinf(eps)) ZZ_FAIL("%s: eps has to be finite and not negative", who);
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    if (!ldr) ldr = D;
    if (!lds) lds = D;
    const int64_t far = (int64_t)1 << 40;
    if ((d_res && (ldr < D || ldr > far)) || (d_sum && (lds < D || lds > far)))
        ZZ_FAIL("%s: rows closer than their width", who);
    if ((uintptr_t)d_res % esz || (uintptr_t)d_sum % esz || (uintptr_t)d_w % 4) ZZ_FAIL("%s: misaligned pointer", who);
    // outputs meet each other and the inputs nowhere, but a sum that is x or res itself
    const int64_t nx = span(ldx, S, D, esz), nr = span(ldr, S, D, esz), nu = span(lds, S, D, esz);
    const int64_t nq = S * zz_fp8_row_bytes(D), ns = (int64_t)zz_f8_nb(D) * S * 4, nw = (int64_t)D * 4;
    const bool own_x = d_sum == d_x && lds == ldx, own_r = d_sum == d_res && lds == ldr;
    int bad = zz_ranges_meet(d_q, nq, d_x, nx) || zz_ranges_meet(d_s, ns, d_x, nx) || zz_ranges_meet(d_q, nq, d_s, ns);
    if (d_res) bad |= zz_ranges_meet(d_q, nq, d_res, nr) || zz_ranges_meet(d_s, ns, d_res, nr);
    if (d_w) bad |= zz_ranges_meet(d_q, nq, d_w, nw) || zz_ranges_meet(d_s, ns, d_w, nw);
    if (d_sum) {
        bad |= zz_ranges_meet(d_q, nq, d_sum, nu) || zz_ranges_meet(d_s, ns, d_sum, nu);
        bad |= !own_x && zz_ranges_meet(d_sum, nu, d_x, nx);
        bad |= d_res && !own_r && zz_ranges_meet(d_sum, nu, d_res, nr);
        bad |= d_w && zz_ranges_meet(d_sum, nu, d_w, nw);
    }
    if (bad) ZZ_FAIL("%s: an output overlaps another argument", who);
    const ZzF8RowsArgs a{d_x, d_res, d_sum, d_w, ldx, ldr, lds, eps, S, D, nu >= ZZ_NT_BYTES, d_q, d_s};
    if (!zz_lib_here(who)) return 0;
    if (!zz_launch_add_norm_fp8(dtype, a, stream ? (hipStream_t)stream : zz_lib_stream()))
        ZZ_FAIL("%s: launch failed", who);
    return 1;
}

extern "C" int zz_rows_fp8_dev(int dtype, const void *d_x, int64_t ldx, int S, int D, uint8_t *d_q, float *d_s,
                               void *stream) {
    const char *who = "zz_rows_fp8_dev";
    if (!rows_common(who, dtype, d_x, &ldx, S, ZZ_F8_MAXP, D, d_q, d_s)) return 0;
    if (D > 1 << 20 || (int64_t)S * zz_f8_nb(D) > 1 << 27) ZZ_FAIL("%s: D <= 2^20, S * ceil(D/128) <= 2^27", who);
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    const int64_t nx = span(ldx, S, D, esz), nq = S * zz_fp8_row_bytes(D), ns = (int64_t)zz_f8_nb(D) * S * 4;
    if (zz_ranges_meet(d_q, nq, d_x, nx) || zz_ranges_meet(d_s, ns, d_x, nx) || zz_ranges_meet(d_q, nq, d_s, ns))
        ZZ_FAIL("%s: an output overlaps another argument", who);
    const ZzF8RowsArgs a{d_x, nullptr, nullptr, nullptr, ldx, 0, 0, 0.0f, S, D, 0, d_q, d_s};
    if (!zz_lib_here(who)) return 0;
    if (!zz_launch_rows_fp8(dtype, a, stream ? (hipStream_t)stream : zz_lib_stream())) ZZ_FAIL("%s: launch failed", who);
    return 1;
}

// ------------------------------------------------------------------ resident matrices
// a table of E matrices [O, I], or of E gated pairs; one plain matrix is a table of one
struct Fp8Mat {
    int E, O, I, parts;             // parts: 1, gated 2
    uint8_t *w = nullptr;           // packed codes (zz_fp8_dev.h), an expert's `wbytes` apart
    float *ws = nullptr;            // [E][parts][ceil(O/128)][ceil(I/128)]
    std::vector<char> loaded;       // [E][parts]
    int missing;                    // of them
};
static std::vector<Fp8Mat *> g_mats;

static size_t wbytes(int O, int I, int parts) {
    const int gc = 32 / parts;      // rows of a matrix in a group of 32
    return (size_t)((O + gc - 1) / gc) * zz_f8_nb(I) * 4096;
}
static size_t wbytes(const Fp8Mat *m) { return wbytes(m->O, m->I, m->parts); }
static size_t scale_count(const Fp8Mat *m) { return (size_t)zz_f8_nb(m->O) * zz_f8_nb(m->I); }

static void free_mat(Fp8Mat *m) {
    if (!m) return;
    zz_lib_mem_bump();
    if (m->w) (void)hipFree(m->w);
    if (m->ws) (void)hipFree(m->ws);
    delete m;
}

static Fp8Mat *get_mat(int id) {
    if (!zz_lib_ready() || id < 0 || id >= (int)g_mats.size()) return nullptr;
    return g_mats[id];
}

static int create(const char *who, int E, int O, int I, int parts) {
    if (!zz_lib_here(who)) return -1;
    size_t id = 0;
    while (id < g_mats.size() && g_mats[id]) id++;
    Fp8Mat *m = nullptr;
    try {
        if (id == g_mats.size()) g_mats.push_back(nullptr);
        m = new Fp8Mat();
        m->loaded.assign((size_t)E * parts, 0);
    } catch (const std::bad_alloc &) {
        delete m;
        zz_set_error("%s: out of memory", who);
        return -1;
    }
    m->E = E;
    m->O = O;
    m->I = I;
    m->parts = parts;
    m->missing = E * parts;
    if (hipMalloc(&m->w, E * wbytes(m)) != hipSuccess ||
        hipMalloc(&m->ws, 4 * E * parts * scale_count(m)) != hipSuccess) {
        (void)hipGetLastError();
        zz_set_error("%s: device allocation failed", who);
        free_mat(m);
        return -1;
    }
    g_mats[id] = m;
    return (int)id;
}

extern "C" int zz_fp8_create(int O, int I) {
    if (O < 1 || O > 1 << 24 || I < 1 || I > 1 << 16 || (int64_t)O * I >= (int64_t)1 << 35) {
        zz_set_error("zz_fp8_create: bad shape (O <= 2^24, I <= 65536, O * I < 2^35)");
        return -1;
    }
    return create("zz_fp8_create", 1, O, I, 1);
}

extern "C" int zz_fp8_create_experts(int E, int O, int I, int gated) {
    const int parts = gated ? 2 : 1;
    if (E < 1 || E > ZZ_F8_MAXE || O < 1 || O > 1 << 24 || I < 1 || I > 1 << 16 || (int64_t)O * I >= (int64_t)1 << 35 ||
        (uint64_t)E * wbytes(O, I, parts) >= (uint64_t)1 << 38) {
        zz_set_error("zz_fp8_create_experts: bad shape (E <= 512, O <= 2^24, I <= 65536, O * I < 2^35, all less than 2^38)");
        return -1;
    }
    return create("zz_fp8_create_experts", E, O, I, parts);
}

extern "C" void zz_fp8_destroy(int id) {
    Fp8Mat *m = get_mat(id);
    if (!m) return;
    (void)hipDeviceSynchronize();
    free_mat(m);
    g_mats[id] = nullptr;
}

// one matrix of the table, from codes on the device and scales there (one launch) or on the host
static int upload_mat(Fp8Mat *m, int e, int part, const uint8_t *d_codes, const float *scales, bool host) {
    hipStream_t st = zz_lib_stream();
    char &have = m->loaded[(size_t)e * m->parts + part];
    m->missing += have;
    have = 0;
    float *ws = m->ws + ((size_t)e * m->parts + part) * scale_count(m);
    if (host) ZZ_CHECK(hipMemcpyAsync(ws, scales, 4 * scale_count(m), hipMemcpyHostToDevice, st));
    if (!zz_launch_fp8_pack(d_codes, m->O, m->I, m->parts == 2 ? part : -1, m->w + e * wbytes(m), host ? nullptr : scales, ws, st))
        ZZ_FAIL("zz_fp8_upload: launch failed");
    ZZ_CHECK(hipStreamSynchronize(st));
    have = 1;
    m->missing--;
    return 1;
}

static int upload_host(const char *who, Fp8Mat *m, int e, int part, const uint8_t *codes, const float *scales) {
    uint8_t *d = nullptr;
    const size_t n = (size_t)m->O * m->I;
    if (hipMalloc(&d, n) != hipSuccess) {
        (void)hipGetLastError();
        ZZ_FAIL("%s: device allocation failed", who);
    }
    const int ok = hipMemcpy(d, codes, n, hipMemcpyHostToDevice) == hipSuccess &&
                   upload_mat(m, e, part, d, scales, true);
    (void)hipFree(d);
    if (!ok) ZZ_FAIL("%s: failed", who);
    return 1;
}

// a matrix that is no table
static Fp8Mat *plain_mat(int id) {
    Fp8Mat *m = get_mat(id);
    return m && m->E == 1 && m->parts == 1 ? m : nullptr;
}

extern "C" int zz_fp8_upload(int id, const uint8_t *codes, const float *scales) {
    if (!codes || !scales) ZZ_FAIL("zz_fp8_upload: bad arguments");
    if (!zz_lib_here("zz_fp8_upload")) return 0;
    Fp8Mat *m = plain_mat(id);
    if (!m) ZZ_FAIL("zz_fp8_upload: no such matrix");
    return upload_host("zz_fp8_upload", m, 0, 0, codes, scales);
}

extern "C" int zz_fp8_upload_dev(int id, const uint8_t *d_codes, const float *d_scales) {
    if (!d_codes || !d_scales || (uintptr_t)d_scales % 4) ZZ_FAIL("zz_fp8_upload_dev: bad arguments");
    if (!zz_lib_here("zz_fp8_upload_dev")) return 0;
    Fp8Mat *m = plain_mat(id);
    if (!m) ZZ_FAIL("zz_fp8_upload_dev: no such matrix");
    return upload_mat(m, 0, 0, d_codes, d_scales, false);
}

static Fp8Mat *expert_mat(const char *who, int id, int e, int part) {
    if (!zz_lib_here(who)) return nullptr;
    Fp8Mat *m = get_mat(id);
    if (m && e >= 0 && e < m->E && part >= 0 && part < m->parts) return m;
    zz_set_error("%s: no such table, expert or part", who);
    return nullptr;
}

extern "C" int zz_fp8_upload_expert(int id, int e, int part, const uint8_t *codes, const float *scales) {
    const char *who = "zz_fp8_upload_expert";
    if (!codes || !scales) ZZ_FAIL("%s: bad arguments", who);
    Fp8Mat *m = expert_mat(who, id, e, part);
    return m ? upload_host(who, m, e, part, codes, scales) : 0;
}

extern "C" int zz_fp8_upload_expert_dev(int id, int e, int part, const uint8_t *d_codes, const float *d_scales) {
    const char *who = "zz_fp8_upload_expert_dev";
    if (!d_codes || !d_scales || (uintptr_t)d_scales % 4) ZZ_FAIL("%s: bad arguments", who);
    Fp8Mat *m = expert_mat(who, id, e, part);
    return m ? upload_mat(m, e, part, d_codes, d_scales, false) : 0;
}

extern "C" int zz_fp8_matmul_dev(int id, const uint8_t *d_q, const float *d_s, int S, int dtype, void *d_y,
                                 int64_t ldy, void *stream) {
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("zz_fp8_matmul_dev: dtype %d declined", dtype);
    if (!d_q || !d_s || !d_y || S < 1 || S > ZZ_F8_MAXS || ldy < 0 || ldy > (int64_t)1 << 40)
        ZZ_FAIL("zz_fp8_matmul_dev: bad arguments (1 <= S <= 2^20)");
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    if ((uintptr_t)d_q % 16 || (uintptr_t)d_s % 4 || (uintptr_t)d_y % esz)
        ZZ_FAIL("zz_fp8_matmul_dev: misaligned pointer");
    if (!zz_lib_here("zz_fp8_matmul_dev")) return 0;
    Fp8Mat *m = plain_mat(id);
    if (!m || m->missing) ZZ_FAIL("zz_fp8_matmul_dev: no such matrix, or it has no weights yet");
    if (!ldy) ldy = m->O;
    if (ldy < m->O) ZZ_FAIL("zz_fp8_matmul_dev: rows of y closer than their width");
    if ((int64_t)S * m->O >= (int64_t)1 << 37) ZZ_FAIL("zz_fp8_matmul_dev: S * O < 2^37");
    const int64_t nq = S * zz_fp8_row_bytes(m->I), ns = (int64_t)zz_f8_nb(m->I) * S * 4, ny = span(ldy, S, m->O, esz);
    if (zz_ranges_meet(d_y, ny, d_q, nq) || zz_ranges_meet(d_y, ny, d_s, ns))
        ZZ_FAIL("zz_fp8_matmul_dev: y overlaps the rows");
    const ZzF8Mat v{m->O, m->I, m->w, m->ws};
    if (!zz_launch_fp8_matmul(v, d_q, d_s, S, dtype, d_y, ldy, stream ? (hipStream_t)stream : zz_lib_stream()))
        ZZ_FAIL("zz_fp8_matmul_dev: launch failed");
    return 1;
}

extern "C" int zz_fp8_matmul(int id, const float *x, float *y, int S) {
    if (!x || !y || S < 1 || S > ZZ_F8_MAXS) ZZ_FAIL("zz_fp8_matmul: bad arguments (1 <= S <= 2^20)");
    if (!zz_lib_here("zz_fp8_matmul")) return 0;
    Fp8Mat *m = plain_mat(id);
    if (!m || m->missing) ZZ_FAIL("zz_fp8_matmul: no such matrix, or it has no weights yet");
    if ((int64_t)S * zz_f8_nb(m->I) > 1 << 27) ZZ_FAIL("zz_fp8_matmul: S * ceil(I/128) <= 2^27");
    hipStream_t st = zz_lib_stream();
    float *dx = nullptr, *ds = nullptr, *dy = nullptr;
    uint8_t *dq = nullptr;
    const size_t nx = (size_t)S * m->I, ny = (size_t)S * m->O;
    const bool mem = hipMalloc(&dx, 4 * nx) == hipSuccess && hipMalloc(&dq, S * zz_fp8_row_bytes(m->I)) == hipSuccess &&
                     hipMalloc(&ds, 4 * (size_t)S * zz_f8_nb(m->I)) == hipSuccess && hipMalloc(&dy, 4 * ny) == hipSuccess;
    if (!mem) {
        (void)hipGetLastError();
        zz_set_error("zz_fp8_matmul: device allocation failed");
    }
    const int ok = mem && hipMemcpyAsync(dx, x, 4 * nx, hipMemcpyHostToDevice, st) == hipSuccess &&
                   zz_rows_fp8_dev(ZZ_F32, dx, 0, S, m->I, dq, ds, st) &&
                   zz_fp8_matmul_dev(id, dq, ds, S, ZZ_F32, dy, 0, st) && hipStreamSynchronize(st) == hipSuccess &&
                   hipMemcpy(y, dy, 4 * ny, hipMemcpyDeviceToHost) == hipSuccess;
    void *ps[] = {dx, dq, ds, dy};
    for (void *p : ps)
        if (p) (void)hipFree(p);
    return ok;                      // the failing step said why
}

// ------------------------------------------------------------------ with an epilogue, and experts
// what both calls check without a device
static int ep_common(const char *who, const ZzF8EpCall &c) {
    if (c.dtype != ZZ_F32 && c.dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, c.dtype);
    const int act = c.act & ~ZZ_EP_8BIT;
    if (act < ZZ_EP_NONE || act > ZZ_EP_SILU) ZZ_FAIL("%s: activation %d declined", who, c.act);
    if (!(c.clamp >= 0.0f) || isinf(c.clamp)) ZZ_FAIL("%s: clamp has to be finite and not negative", who);
    const int64_t far = (int64_t)1 << 36;                 // P rows' bytes stay under 2^62
    if (!c.q || !c.s || !c.y || c.ldy < 0 || c.ldy > far || c.ldr < 0 || c.ldr > far) ZZ_FAIL("%s: bad arguments", who);
    const int esz = c.dtype == ZZ_F32 ? 4 : 2;
    if ((uintptr_t)c.q % 16 || (uintptr_t)c.s % 4 || (uintptr_t)c.y % esz || (uintptr_t)c.res % esz ||
        (uintptr_t)c.bias % 4 || (uintptr_t)c.row % 4 || (uintptr_t)c.offs % 4)
        ZZ_FAIL("%s: misaligned pointer", who);
    return 1;
}

static int ep_run(const char *who, Fp8Mat *m, ZzF8EpCall &c, void *stream) {
    const int esz = c.dtype == ZZ_F32 ? 4 : 2, nb = zz_f8_nb(m->I);
    if (m->parts == 1 && c.clamp > 0.0f) ZZ_FAIL("%s: a clamp is a gated pair's", who);
    if (!c.ldy) c.ldy = m->O;
    if (!c.ldr) c.ldr = m->O;
    if (c.ldy < m->O || (c.res && c.ldr < m->O)) ZZ_FAIL("%s: rows closer than their width", who);
    if ((int64_t)c.P * m->O >= (int64_t)1 << 37) ZZ_FAIL("%s: results of 2^37 elements or more", who);
    if (!zz_f8_ep_fits(m->parts * m->O, c.P, c.E, c.offs != nullptr))
        ZZ_FAIL("%s: results of 2^24 tiles or more (128 rows, %d columns)", who, 128 / m->parts);
    if (c.row && (uint64_t)c.R * zz_fp8_row_bytes(m->I) >= (uint64_t)1 << 32)
        ZZ_FAIL("%s: rows by index within 2^32 bytes", who);
    const int64_t ny = span(c.ldy, c.P, m->O, esz);
    const bool own = c.res == c.y && c.ldr == c.ldy;
    int bad = zz_ranges_meet(c.y, ny, c.q, c.R * zz_fp8_row_bytes(m->I)) || zz_ranges_meet(c.y, ny, c.s, (int64_t)nb * c.R * 4);
    if (c.bias) bad |= zz_ranges_meet(c.y, ny, c.bias, (int64_t)c.E * m->parts * m->O * 4);
    if (c.res && !own) bad |= zz_ranges_meet(c.y, ny, c.res, span(c.ldr, c.P, m->O, esz));
    if (c.row) bad |= zz_ranges_meet(c.y, ny, c.row, (int64_t)c.P * 4);
    if (c.offs) bad |= zz_ranges_meet(c.y, ny, c.offs, (int64_t)(c.E + 1) * 4);
    if (bad) ZZ_FAIL("%s: y overlaps another argument", who);
    c.m = ZzF8Mat{m->O, m->I, m->w, m->ws};
    c.we = (int64_t)wbytes(m);
    c.wsu = (int)scale_count(m);
    c.wse = m->parts * c.wsu;
    c.eight = c.act & ZZ_EP_8BIT;
    c.act &= ~ZZ_EP_8BIT;
    hipStream_t st = stream ? (hipStream_t)stream : zz_lib_stream();
    if (!(m->parts == 2 ? zz_launch_fp8_gated(c, st) : zz_launch_fp8_ep(c, st))) ZZ_FAIL("%s: launch failed", who);
    return 1;
}

extern "C" int zz_fp8_matmul_ep_dev(int id, const uint8_t *d_q, const float *d_s, int S, const float *d_bias, int act,
                                    float clamp, const void *d_res, int64_t ldr, int dtype, void *d_y, int64_t ldy,
                                    void *stream) {
    const char *who = "zz_fp8_matmul_ep_dev";
    ZzF8EpCall c{};
    c.q = d_q; c.s = d_s; c.R = c.P = S; c.E = 1; c.bias = d_bias; c.res = d_res; c.ldr = ldr; c.act = act;
    c.clamp = clamp; c.dtype = dtype; c.y = d_y; c.ldy = ldy;
    if (!ep_common(who, c)) return 0;
    if (S < 1 || S > ZZ_F8_MAXS) ZZ_FAIL("%s: bad arguments (1 <= S <= 2^20)", who);
    if (!zz_lib_here(who)) return 0;
    Fp8Mat *m = get_mat(id);
    if (!m || m->E != 1 || m->missing) ZZ_FAIL("%s: no such matrix, or it has no weights yet", who);
    return ep_run(who, m, c, stream);
}

extern "C" int zz_fp8_matmul_experts_dev(int id, const uint8_t *d_q, const float *d_s, int R, const int *d_row,
                                         const int *d_offs, int P, const float *d_bias, int act, float clamp,
                                         const void *d_res, int64_t ldr, int dtype, void *d_y, int64_t ldy,
                                         void *stream) {
    const char *who = "zz_fp8_matmul_experts_dev";
    ZzF8EpCall c{};
    c.q = d_q; c.s = d_s; c.R = R; c.P = P; c.row = d_row; c.offs = d_offs; c.bias = d_bias; c.res = d_res;
    c.ldr = ldr; c.act = act; c.clamp = clamp; c.dtype = dtype; c.y = d_y; c.ldy = ldy;
    if (!ep_common(who, c)) return 0;
    if (!d_offs || P < 1 || P > ZZ_F8_MAXP || R < 1 || R > ZZ_F8_MAXP) ZZ_FAIL("%s: bad arguments (1 <= P, R <= 2^24)", who);
    if (!d_row && R < P) ZZ_FAIL("%s: without an index R >= P", who);
    if (!zz_lib_here(who)) return 0;
    Fp8Mat *m = get_mat(id);
    if (!m || m->missing) ZZ_FAIL("%s: no such table, or it has experts without weights", who);
    c.E = m->E;
    return ep_run(who, m, c, stream);
}

// released by gpu_shutdown (zz_api.hip)
void zz_fp8_shutdown() {
    for (Fp8Mat *&m : g_mats) { free_mat(m); m = nullptr; }
    g_mats.clear();
}
