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

static int rows_common(const char *who, int dtype, const void *x, int64_t *ldx, int S, int D, const uint8_t *q,
                       const float *s) {
    if (dtype != ZZ_F32 && dtype != ZZ_BF16) ZZ_FAIL("%s: dtype %d declined", who, dtype);
    if (!x || !q || !s || S < 1 || S > ZZ_F8_MAXS || D < 1) ZZ_FAIL("%s: bad arguments (1 <= S <= 2^20)", who);
    if (!*ldx) *ldx = D;
    if (*ldx < D || *ldx > (int64_t)1 << 40) ZZ_FAIL("%s: rows closer than their width", who);
    const int esz = dtype == ZZ_F32 ? 4 : 2;
    if ((uintptr_t)x % esz || (uintptr_t)q % 16 || (uintptr_t)s % 4) ZZ_FAIL("%s: misaligned pointer", who);
    return 1;
}

static int64_t span(int64_t ld, int S, int D, int esz) { return ((S - 1) * ld + D) * esz; }

extern "C" int zz_add_norm_fp8_dev(int dtype, const void *d_x, int64_t ldx, const void *d_res, int64_t ldr,
                                   void *d_sum, int64_t lds, const float *d_w, float eps, int S, int D,
                                   uint8_t *d_q, float *d_s, void *stream) {
    const char *who = "zz_add_norm_fp8_dev";
    if (!rows_common(who, dtype, d_x, &ldx, S, D, d_q, d_s)) return 0;
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
    if (!rows_common(who, dtype, d_x, &ldx, S, D, d_q, d_s)) return 0;
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
struct Fp8Mat {
    int O, I;
    uint8_t *w = nullptr;           // packed codes (zz_fp8_dev.h)
    float *ws = nullptr;
    bool loaded = false;
};
static std::vector<Fp8Mat *> g_mats;

static size_t packed_bytes(const Fp8Mat *m) { return (size_t)((m->O + 31) / 32) * zz_f8_nb(m->I) * 4096; }
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

extern "C" int zz_fp8_create(int O, int I) {
    if (O < 1 || O > 1 << 24 || I < 1 || I > 1 << 16 || (int64_t)O * I >= (int64_t)1 << 35) {
        zz_set_error("zz_fp8_create: bad shape (O <= 2^24, I <= 65536, O * I < 2^35)");
        return -1;
    }
    if (!zz_lib_here("zz_fp8_create")) return -1;
    size_t id = 0;
    while (id < g_mats.size() && g_mats[id]) id++;
    Fp8Mat *m = nullptr;
    try {
        if (id == g_mats.size()) g_mats.push_back(nullptr);
        m = new Fp8Mat();
    } catch (const std::bad_alloc &) {
        zz_set_error("zz_fp8_create: out of memory");
        return -1;
    }
    m->O = O;
    m->I = I;
    if (hipMalloc(&m->w, packed_bytes(m)) != hipSuccess || hipMalloc(&m->ws, 4 * scale_count(m)) != hipSuccess) {
        (void)hipGetLastError();
        zz_set_error("zz_fp8_create: device allocation failed");
        free_mat(m);
        return -1;
    }
    g_mats[id] = m;
    return (int)id;
}

extern "C" void zz_fp8_destroy(int id) {
    Fp8Mat *m = get_mat(id);
    if (!m) return;
    (void)hipDeviceSynchronize();
    free_mat(m);
    g_mats[id] = nullptr;
}

static int upload_mat(Fp8Mat *m, const uint8_t *d_codes, const void *scales, hipMemcpyKind kind) {
    hipStream_t st = zz_lib_stream();
    m->loaded = false;
    ZZ_CHECK(hipMemcpyAsync(m->ws, scales, 4 * scale_count(m), kind, st));
    if (!zz_launch_fp8_pack(d_codes, m->O, m->I, m->w, st)) ZZ_FAIL("zz_fp8_upload: launch failed");
    ZZ_CHECK(hipStreamSynchronize(st));
    m->loaded = true;
    return 1;
}

extern "C" int zz_fp8_upload(int id, const uint8_t *codes, const float *scales) {
    if (!codes || !scales) ZZ_FAIL("zz_fp8_upload: bad arguments");
    if (!zz_lib_here("zz_fp8_upload")) return 0;
    Fp8Mat *m = get_mat(id);
    if (!m) ZZ_FAIL("zz_fp8_upload: no such matrix");
    uint8_t *d = nullptr;
    const size_t n = (size_t)m->O * m->I;
    if (hipMalloc(&d, n) != hipSuccess) {
        (void)hipGetLastError();
        ZZ_FAIL("zz_fp8_upload: device allocation failed");
    }
    const int ok = hipMemcpy(d, codes, n, hipMemcpyHostToDevice) == hipSuccess &&
                   upload_mat(m, d, scales, hipMemcpyHostToDevice);
    (void)hipFree(d);
    if (!ok) ZZ_FAIL("zz_fp8_upload: failed");
    return 1;
}

extern "C" int zz_fp8_upload_dev(int id, const uint8_t *d_codes, const float *d_scales) {
    if (!d_codes || !d_scales || (uintptr_t)d_scales % 4) ZZ_FAIL("zz_fp8_upload_dev: bad arguments");
    if (!zz_lib_here("zz_fp8_upload_dev")) return 0;
    Fp8Mat *m = get_mat(id);
    if (!m) ZZ_FAIL("zz_fp8_upload_dev: no such matrix");
    return upload_mat(m, d_codes, d_scales, hipMemcpyDeviceToDevice);
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
    Fp8Mat *m = get_mat(id);
    if (!m || !m->loaded) ZZ_FAIL("zz_fp8_matmul_dev: no such matrix, or it has no weights yet");
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
    Fp8Mat *m = get_mat(id);
    if (!m || !m->loaded) ZZ_FAIL("zz_fp8_matmul: no such matrix, or it has no weights yet");
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

// released by gpu_shutdown (zz_api.hip)
void zz_fp8_shutdown() {
    for (Fp8Mat *&m : g_mats) { free_mat(m); m = nullptr; }
    g_mats.clear();
}
