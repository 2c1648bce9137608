// psfm_linear.hip — the pointwise product's entry points (include/psfm_linear.h): argument checks, the choice
// of tiles and splits, workspaces.  The kernels are in psfm_linear_kernels.h.
#include "psfm_linear.h"

#include <algorithm>
#include <string>

using namespace psfm;

namespace {

thread_local std::string g_err;

int fail(int code, const char* msg) {
    g_err = msg;
    return code;
}
int status(int e, const char* what) {
    if (e == 0) return 0;
    g_err = std::string(what) + ": " + hipGetErrorString((hipError_t)e);
    return e;
}

constexpr int64_t MAX_DIM = (int64_t)1 << 40;

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t size_of(int dtype) { return dtype == PSFM_DTYPE_F32 ? 4 : 2; }
const LinearOps& ops_of(int dtype) {
    return dtype == PSFM_DTYPE_F32 ? linear_ops_f32() : dtype == PSFM_DTYPE_F16 ? linear_ops_f16() : linear_ops_bf16();
}

int check(const psfm_linear* d) {
    if (!d) return fail(-1, "psfm_linear: no descriptor");
    if (d->M < 0 || d->N < 0 || d->K < 0 || d->M > MAX_DIM || d->N > MAX_DIM || d->K > MAX_DIM)
        return fail(-2, "psfm_linear: M, N and K must be 0 .. 2^40");
    const double most = 4.6e18;   // values and byte offsets fit 63 bits
    if ((double)d->M * (double)d->N * 4 > most || (double)d->N * (double)d->K * 4 > most || d->ldx < d->K ||
        d->ldr < 0 || (double)d->M * (double)d->ldx * 4 > most || (double)d->M * (double)d->ldr * 4 > most)
        return fail(-3, "psfm_linear: a row stride below the row's length, or a size over 63 bits");
    if (d->dtype != PSFM_DTYPE_F32 && d->dtype != PSFM_DTYPE_F16 && d->dtype != PSFM_DTYPE_BF16)
        return fail(-4, "psfm_linear: dtype must be PSFM_DTYPE_F32 / F16 / BF16");
    if (d->act < PSFM_ACT_NONE || d->act > PSFM_ACT_GELU) return fail(-5, "psfm_linear: unknown activation");
    if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(-6, "psfm_linear: p must be in 0 .. 1");
    if (d->p > 0.0 && (!d->rng || d->mask_rows < 1)) return fail(-7, "psfm_linear: dropout needs rng and mask_rows >= 1");
    return 0;
}

DropArgs drop_of(const psfm_linear* d) {
    DropArgs a{nullptr, 0, 1.0f, 1};
    if (d->p > 0.0 && drop_threshold(d->p, &a.last, &a.scale)) a.rng = d->rng, a.mask_rows = d->mask_rows;
    return a;
}

struct Plan {
    int variant;
    int64_t ti, tj, rsplit;
    int splits;
    int64_t blocks() const { return ti * tj * splits; }
};

// Tiles: the large one once it fills the 256 CUs, else the small one.  The reduction is split while the tiles
// alone leave CUs idle and a split keeps at least four LDS stages.
Plan plan(int dtype, int64_t I, int64_t J, int64_t R) {
    Plan p{0, 0, 0, 0, 1};
    for (int v = LINEAR_NTILES - 1; v >= 0; --v) {
        p.variant = v, p.ti = up(I, LINEAR_TILES[v].bi), p.tj = up(J, LINEAR_TILES[v].bj);
        if (p.ti * p.tj >= 256) break;
    }
    const int64_t stage = 128 / size_of(dtype), stages = up(R, stage), tiles = p.ti * p.tj;
    int64_t splits = 1;
    if (tiles > 0 && tiles < 256) splits = std::max<int64_t>(1, std::min(up(512, tiles), stages / 4));
    const int64_t per = std::max<int64_t>(1, up(stages, splits));
    p.rsplit = per * stage;
    p.splits = (int)std::max<int64_t>(1, up(stages, per));
    return p;
}

int64_t part_bytes(const Plan& p, int64_t I, int64_t J) { return p.splits > 1 ? p.splits * I * J * 4 : 0; }
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct DzPlan {
    int64_t gx, gy, rows;
};
// About four workgroups a CU, each with a few rows a thread at least.
DzPlan dz_plan(int dtype, int64_t M, int64_t N) {
    DzPlan p;
    const int64_t v = 16 / size_of(dtype), cb = N <= DZ_NARROW * v ? DZ_NARROW : DZ_WIDE, rp = DZ_THREADS / cb;
    p.gx = up(N, cb * v);
    p.gy = std::max<int64_t>(1, std::min(up(1024, std::max<int64_t>(p.gx, 1)), up(M, 2 * rp)));
    p.rows = up(std::max<int64_t>(M, 1), p.gy);
    p.gy = up(std::max<int64_t>(M, 1), p.rows);
    return p;
}

bool mult(const void* p, int64_t ld, int64_t edge, int64_t v) {
    return ((uintptr_t)p & 15) == 0 && ld % v == 0 && edge % v == 0;
}

int run_gemm(int role, int dtype, GemmArgs& a, const Plan& p, void* ws, hipStream_t s) {
    const int64_t v = 16 / size_of(dtype);
    const bool pt = role == GEMM_DW, qt = role != GEMM_FWD;
    const bool vec = mult(a.P, a.ldp, pt ? a.I : a.R, v) && mult(a.Q, a.ldq, qt ? a.J : a.R, v);
    if (p.blocks() > 0x7fffffff) return fail(-8, "psfm_linear: more tiles than a launch holds");
    a.ti = (uint32_t)p.ti, a.tj = (uint32_t)p.tj, a.splits = p.splits, a.rsplit = p.rsplit, a.part = (float*)ws;
    const LinearOps& o = ops_of(dtype);
    int e = o.gemm(role, p.variant, vec, a, s);
    if (e == 0 && p.splits > 1) e = o.join(a, role == GEMM_FWD, s);
    return status(e, "psfm_linear: launch");
}

struct BwdPlan {
    bool dz;          // dz has to be made (an activation or a mask); else it is dy
    int64_t dz_at, cols_at, parts_at, bytes;
    Plan dx, dw;
    DzPlan cols;
};
BwdPlan bwd_plan(const psfm_linear* d, bool want_dx, bool want_dw, bool want_db) {
    BwdPlan b{};
    b.dz = (want_dx || want_dw) && (d->act != PSFM_ACT_NONE || drop_of(d).rng);
    b.cols = dz_plan(d->dtype, d->M, d->N);
    b.dz_at = 0;
    b.cols_at = b.dz ? aligned(d->M * d->N * size_of(d->dtype)) : 0;
    b.parts_at = b.cols_at + (want_db ? aligned(b.cols.gy * d->N * 4) : 0);
    int64_t parts = 0;
    if (want_dx) b.dx = plan(d->dtype, d->M, d->K, d->N), parts = std::max(parts, part_bytes(b.dx, d->M, d->K));
    if (want_dw) b.dw = plan(d->dtype, d->N, d->K, d->M), parts = std::max(parts, part_bytes(b.dw, d->N, d->K));
    b.bytes = b.parts_at + parts;
    return b;
}

}  // namespace

extern "C" {

int64_t psfm_linear_fwd_ws_bytes(const psfm_linear* d) {
    if (check(d)) return -1;
    return part_bytes(plan(d->dtype, d->M, d->N, d->K), d->M, d->N);
}

int psfm_linear_fwd(const psfm_linear* d, const void* x, const void* w, const void* bias, const void* res, void* y,
                    void* z, void* ws, void* stream) {
    if (const int rc = check(d)) return rc;
    if (d->M == 0 || d->N == 0) return 0;
    if (!y || (d->K > 0 && (!x || !w))) return fail(-9, "psfm_linear_fwd: null tensor");
    if (res && d->ldr < d->N) return fail(-3, "psfm_linear_fwd: ldr below N");
    const Plan p = plan(d->dtype, d->M, d->N, d->K);
    if (part_bytes(p, d->M, d->N) > 0 && !ws) return fail(-10, "psfm_linear_fwd: no workspace");
    GemmArgs a{};
    a.P = x, a.Q = w, a.ldp = d->ldx, a.ldq = d->K, a.I = d->M, a.J = d->N, a.R = d->K;
    a.e = LinearEpi{y, bias, res, d->ldr, z, d->act, 1.0f, drop_of(d)};
    return run_gemm(GEMM_FWD, d->dtype, a, p, ws, (hipStream_t)stream);
}

int64_t psfm_linear_bwd_ws_bytes(const psfm_linear* d, int want_dx, int want_dw, int want_db) {
    if (check(d)) return -1;
    return bwd_plan(d, want_dx, want_dw, want_db).bytes;
}

int psfm_linear_bwd(const psfm_linear* d, const void* dy, const void* x, const void* w, const void* z, void* dx,
                    void* dw, void* db, void* ws, void* stream) {
    if (const int rc = check(d)) return rc;
    const bool any = d->M > 0 && d->N > 0;
    if (any && (!dy || (d->act != PSFM_ACT_NONE && !z) || (dx && d->K > 0 && !w) || (dw && d->K > 0 && !x)))
        return fail(-9, "psfm_linear_bwd: null tensor");
    const BwdPlan b = bwd_plan(d, dx, dw, db);
    if (b.bytes > 0 && !ws) return fail(-10, "psfm_linear_bwd: no workspace");
    if (b.cols.gx > 0x7fffffff) return fail(-8, "psfm_linear_bwd: more columns than a launch holds");
    const hipStream_t s = (hipStream_t)stream;
    const LinearOps& o = ops_of(d->dtype);
    const DropArgs drop = drop_of(d);
    float* cols = (float*)((char*)ws + b.cols_at);
    const void* dz = b.dz ? ws : dy;
    if (any && (b.dz || db)) {
        const DzArgs a{dy, d->act != PSFM_ACT_NONE ? z : nullptr, b.dz ? ws : nullptr, db ? cols : nullptr,
                       d->M, d->N, b.cols.rows, d->act, drop};
        if (const int rc = status(o.dz(a, b.cols.gx, b.cols.gy, s), "psfm_linear_bwd: dz launch")) return rc;
    }
    if (db && d->N > 0) {
        const int e = o.colsum(cols, any ? b.cols.gy : 0, d->N, drop.scale, db, s);
        if (const int rc = status(e, "psfm_linear_bwd: column sums launch")) return rc;
    }
    void* parts = (char*)ws + b.parts_at;
    if (dx && d->M > 0 && d->K > 0) {
        GemmArgs a{};
        a.P = dz, a.Q = w, a.ldp = d->N, a.ldq = d->K, a.I = d->M, a.J = d->K, a.R = d->N;
        a.e.out = dx, a.e.alpha = drop.scale;
        if (const int rc = run_gemm(GEMM_DX, d->dtype, a, b.dx, parts, s)) return rc;
    }
    if (dw && d->N > 0 && d->K > 0) {
        GemmArgs a{};
        a.P = dz, a.Q = x, a.ldp = d->N, a.ldq = d->ldx, a.I = d->N, a.J = d->K, a.R = d->M;
        a.e.out = dw, a.e.alpha = drop.scale;
        if (const int rc = run_gemm(GEMM_DW, d->dtype, a, b.dw, parts, s)) return rc;
    }
    return 0;
}

const char* psfm_linear_last_error(void) { return g_err.c_str(); }

}  // extern "C"
