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
    double alone, busy, join;   // estimates: the larger of the first two, and the join
    int64_t blocks() const { return ti * tj * splits; }
    bool fits() const { return blocks() <= most_blocks(LINEAR_TILES[variant].threads); }
};

// The tile and the splits of the reduction that should take least time, from what a stage of 128 bytes of reduction
// takes (us): `alone` where a CU has one or two workgroups and waits for memory, `busy` per workgroup where it
// has enough of them, and from `out`, a tile's way through the forward epilogue (short reductions live from small tiles: 50000 x
// 256 over 64 in bf16 14.3, 17.9 and 18.5 us in tiles of 64, 128 and 256; over 1024 44.4, 41.9, 41.0); splits write no
// tile but add a launch and their way through memory.  From a sweep of every tile and 1 .. 16
// splits over products from 300 x 500 x 1200 to 16384 x 1024 x 256 (I x J x R); the choice was within a seventh of the best
// one (bf16 1024 x 1024 x 1024: 8.0 us as chosen, 64 tiles in one piece; two pieces 13.8; 128 tiles 16.7; 256 tiles 33.
// 256 x 1024 x 4096: 11.1 in four pieces, 12.2 in two.  512 x 4096 x 4096: 26.9, 128 tiles in four pieces 31.3).  Rows that
// are no whole chunks go through registers, and wait for memory half as long again.  STAGED: dz made on the way, whose
// every stage waits for its loads and the activation's slope (8192 x 2048, reduction 128 in bf16: 41 us in 16 pieces, 42 in
// 8, 220 in one).  It is one cost for all: measured with a slope and dz's rest, too high for ReLU and for none, which have neither.
struct TileTime {
    double alone, busy, out;
};
constexpr TileTime TIMES16[] = {{0.42, 0.22, 0.4}, {1.15, 0.5, 3.4}, {2.0, 2.0, 13.0}},
                   TIMES32[] = {{0.8, 0.61, 0.5}, {2.4, 2.39, 3.0}}, STAGED16[] = {{1.75, 1.15, 0}},
                   STAGED32[] = {{1.45, 1.0, 0}};

bool chunks(const psfm_linear* d) {
    const int64_t v = 16 / size_of(d->dtype);
    return d->N % v == 0 && d->K % v == 0 && d->ldx % v == 0;
}

Plan plan(const psfm_linear* d, int64_t I, int64_t J, int64_t R, bool forward, int largest = LINEAR_NTILES - 1,
          bool staged = false) {
    static const int SPLITS[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256, 384, 512};
    const bool wide = d->dtype == PSFM_DTYPE_F32;
    const TileTime* times = staged ? (wide ? STAGED32 : STAGED16) : wide ? TIMES32 : TIMES16;
    const int64_t stage = 128 / size_of(d->dtype), stages = up(R, stage);
    const double wait = chunks(d) ? 1.0 : 1.5;
    Plan best{0, 0, 0, 0, 1, 0, 0, 0};
    double least = 0;
    for (int v = staged ? 0 : std::min(largest, wide ? 1 : 2); v >= 0; --v) {
        const int64_t ti = up(I, LINEAR_TILES[v].bi), tj = up(J, LINEAR_TILES[v].bj);
        for (const int want : SPLITS) {
            const int64_t per = std::max<int64_t>(1, up(stages, want)), n = std::max<int64_t>(1, up(stages, per));
            if (want > 1 && (per < 2 || ti * tj * n > 4096)) break;
            if (ti * tj * n > most_blocks(LINEAR_TILES[v].threads)) break;
            const double blocks = (double)ti * (double)tj * (double)n, load = staged ? 1.0 : std::min(1.0, blocks / 512);
            const double rounds = (double)up((int64_t)std::min(blocks, 1e15), 256), out = forward && n == 1 ? times[v].out : 0.0;
            const double alone = (double)per * times[v].alone * wait * (0.64 + 0.36 * load) + out;
            const double busy = ((double)per * times[v].busy + out) * rounds;
            const double join = n == 1 ? 0.0 : 4.0 + 0.15 * (double)std::min<int64_t>(n, 8) + 0.012 * (double)n +
                                                   (double)n * (double)I * (double)J * 8 / 5e6;
            const double t = std::max(alone, busy) + join;
            if (best.rsplit == 0 || t < least) least = t, best = Plan{v, ti, tj, per * stage, (int)n, alone, busy, join};
        }
    }
    if (best.rsplit == 0) {   // no launch holds it: the caller finds that it does not fit
        const int v = staged ? 0 : std::min(largest, wide ? 1 : 2);
        best = Plan{v, up(I, LINEAR_TILES[v].bi), up(J, LINEAR_TILES[v].bj), std::max<int64_t>(1, stages) * stage, 1, 1e30, 1e30, 0};
    }
    return best;
}

int64_t part_bytes(const Plan& p, int64_t I, int64_t J) { return p.splits > 1 ? p.splits * I * J * 4 : 0; }
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }
bool mult(const void* p, int64_t ld, int64_t edge, int64_t v) {
    return ((uintptr_t)p & 15) == 0 && ld % v == 0 && edge % v == 0;
}

// Rows that one matrix instruction takes, or two where W's rows are short.  4096 x 4096 bf16, 16 rows: 9.9 us, 10.2 in
// tiles; 32 rows: 13.6, 11.2.  1024 x 1024, 32 rows: 5.1, 6.5.  fp32 4096 x 4096, 16 rows: 20.1, 27.0; 32 rows: 28.9,
// 27.8; 512 x 512, 32 rows: 6.2, 7.9.
bool skinny(const psfm_linear* d) {
    return (d->M <= 16 || (d->M <= SKINNY_ROWS && d->K * size_of(d->dtype) < 4096)) && up(d->N, 16) <= most_blocks(SKINNY_THREADS);
}

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

struct BwdPlan {
    bool dx, dw;       // products to take (a wanted gradient of no values is none)
    bool stage;        // the products make dz from dy as they stage it
    bool pass;         // dz, or the column sums alone, as a pass of its own
    bool dz;           // ... which writes dz
    int64_t parts;     // of the column sums (0: the product writes db itself)
    int64_t cols_at, dxp_at, dwp_at, bytes;
    Plan pdx, pdw;
    DzPlan cols;
};

// The time of the products together: they share a launch where they share a tile.
double together(const BwdPlan& b) {
    const Plan none{}, &x = b.dx ? b.pdx : none, &w = b.dw ? b.pdw : none;
    if (x.variant != w.variant) return std::max(x.alone, x.busy) + std::max(w.alone, w.busy) + std::max(x.join, w.join);
    return std::max({x.alone, w.alone, x.busy + w.busy}) + std::max(x.join, w.join);
}

constexpr int64_t FEW_DZ = 1 << 15;

// The products make dz themselves, in the smallest tiles, where that should take less time than a pass of its own, a launch
// and dz's way to memory and back.  bf16, both gradients and the bias's, replayed in a graph (rows x K x N): 64 x 4096 x 64 5.2 us,
// 8.3 with a pass; 480 x 64 x 64 9.5, 10.9; 480 x 512 x 256 13.8, 11.9; 184320 x 128 x 64 64, 51; 8192 x 256 x 2048 126, 52.
// fp32: 480 x 64 x 256 10.2, 15.8; 30720 x 128 x 64 29, 35; 184320 x 256 x 64 195, 177; 8192 x 256 x 2048 242, 186.  A pass
// rounds dz to the type once more, 16 bits off by up to sqrt(2) of one rounding where that averages over many values; with
// few of them (1.49 was seen at 1500) the products make it for some microseconds more too.  (fp16, either way: a dz below 2^-25 is lost, one
// beyond 65504 infinite; no scale is safe for all of dy's range.)  The choice is the layer's, for all gradients together: what dx and dw are
// does not depend on which others are asked for (db sums its rows in another order where no dw is made beside it).
BwdPlan bwd_plan(const psfm_linear* d, bool want_dx, bool want_dw, bool want_db) {
    BwdPlan b{};
    const bool any = d->M > 0 && d->N > 0, make = d->act != PSFM_ACT_NONE || drop_of(d).rng;
    b.dx = b.dw = any && d->K > 0;
    // turned operands of odd rows leave the largest tile no registers (8191 x 1023 over 8191, bf16: 636 us, 172 in the next one)
    const int largest = chunks(d) ? LINEAR_NTILES - 1 : 1;
    auto plans = [&](bool staged) {
        if (d->M > 0 && d->K > 0) b.pdx = plan(d, d->M, d->K, d->N, false, largest, staged);
        if (d->N > 0 && d->K > 0) b.pdw = plan(d, d->N, d->K, d->M, false, largest, staged);
        return together(b);
    };
    const double moved = (double)d->M * (double)d->N * size_of(d->dtype) * (2 + (d->act != PSFM_ACT_NONE));
    const double few = size_of(d->dtype) == 2 && d->M * d->N < FEW_DZ ? 4.0 : 0.0;
    b.stage = make && b.dx && plans(true) < plans(false) + 5.5 + few + moved / 5e6;
    plans(b.stage);
    b.dx = want_dx && d->M > 0 && d->K > 0;
    b.dw = want_dw && d->N > 0 && d->K > 0;
    b.stage = b.stage && (b.dx || b.dw);
    b.dz = make && !b.stage && any && (b.dx || b.dw);
    b.pass = b.dz || (want_db && any && !(b.stage && b.dw));   // the latter: the column sums alone
    b.cols = dz_plan(d->dtype, d->M, d->N);
    b.parts = !want_db || !any ? 0 : b.pass ? b.cols.gy : b.pdw.splits > 1 ? b.pdw.splits : 0;
    b.cols_at = b.dz ? aligned(d->M * d->N * size_of(d->dtype)) : 0;
    b.dxp_at = b.cols_at + aligned(b.parts * d->N * 4);
    b.dwp_at = b.dxp_at + (b.dx ? aligned(part_bytes(b.pdx, d->M, d->K)) : 0);
    b.bytes = b.dwp_at + (b.dw ? part_bytes(b.pdw, d->N, d->K) : 0);
    return b;
}

// whole chunks at other addresses: the next tile, whose splits are the same
void retile(Plan& p, int64_t I, int64_t J) {
    if (p.variant < 2) return;
    p.variant = 1, p.ti = up(I, LINEAR_TILES[1].bi), p.tj = up(J, LINEAR_TILES[1].bj);
}

void set(GemmArgs& a, const Plan& p, void* parts) {
    a.ti = (uint32_t)p.ti, a.tj = (uint32_t)p.tj, a.splits = p.splits, a.rsplit = p.rsplit, a.part = (float*)parts;
}

}  // namespace

extern "C" {

int64_t psfm_linear_fwd_ws_bytes(const psfm_linear* d) {
    if (check(d)) return -1;
    return skinny(d) ? 0 : part_bytes(plan(d, d->M, d->N, d->K, true), d->M, d->N);
}

int psfm_linear_fwd(const psfm_linear* d, const void* x, const void* w, const void* bias, const void* res, void* y,
                    void* z, void* ws, void* stream) {
    if (const int rc = check(d)) return rc;
    if (d->M == 0 || d->N == 0) return 0;
    if (!y || (d->K > 0 && (!x || !w))) return fail(-9, "psfm_linear_fwd: null tensor");
    if (res && d->ldr < d->N) return fail(-3, "psfm_linear_fwd: ldr below N");
    const LinearOps& o = ops_of(d->dtype);
    const hipStream_t s = (hipStream_t)stream;
    const LinearEpi e{y, bias, res, d->ldr, z, d->act, 1.0f, drop_of(d)};
    const int64_t v = 16 / size_of(d->dtype);
    const bool vec = mult(x, d->ldx, d->K, v) && mult(w, d->K, d->K, v);
    if (skinny(d))
        return status(o.skinny(vec, SkinnyArgs{x, w, d->ldx, d->M, d->N, d->K, e}, s), "psfm_linear_fwd: launch");
    const Plan p = plan(d, d->M, d->N, d->K, true);
    if (p.splits > 1 && !ws) return fail(-10, "psfm_linear_fwd: no workspace");
    if (!p.fits()) return fail(-8, "psfm_linear_fwd: more tiles than a launch holds");
    GemmArgs a{};
    a.P = x, a.Q = w, a.ldp = d->ldx, a.ldq = d->K, a.I = d->M, a.J = d->N, a.R = d->K, a.e = e;
    set(a, p, ws);
    int rc = o.forward(p.variant, vec, a, s);
    if (rc == 0 && p.splits > 1) rc = o.join(a, s);
    return status(rc, "psfm_linear_fwd: launch");
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
    BwdPlan b = bwd_plan(d, dx, dw, db);
    if (b.bytes > 0 && !ws) return fail(-10, "psfm_linear_bwd: no workspace");
    const void* dz = b.dz ? ws : dy;
    const int64_t v = 16 / size_of(d->dtype);
    const bool vec = d->N % v == 0 && d->K % v == 0 && ((uintptr_t)dz & 15) == 0 &&
                     (!b.stage || d->act == PSFM_ACT_NONE || ((uintptr_t)z & 15) == 0) &&
                     (!b.dx || ((uintptr_t)w & 15) == 0) && (!b.dw || mult(x, d->ldx, d->K, v));
    if (!vec) retile(b.pdx, d->M, d->K), retile(b.pdw, d->N, d->K);
    // k_finish: 16 columns of db a workgroup, and the joins, whose products have at most 4096 tiles (plan): under 2^19 each
    if ((b.pass && b.cols.gx > most_blocks(DZ_THREADS)) || (b.dx && !b.pdx.fits()) || (b.dw && !b.pdw.fits()) ||
        (db && up(d->N, 16) + (1 << 20) > most_blocks(FINISH_THREADS)))
        return fail(-8, "psfm_linear_bwd: more tiles or columns than a launch holds");
    const hipStream_t s = (hipStream_t)stream;
    const LinearOps& o = ops_of(d->dtype);
    const DropArgs drop = drop_of(d);
    const DzArgs make{d->act != PSFM_ACT_NONE ? z : nullptr, d->act, drop, nullptr, nullptr};
    char* at = (char*)ws;
    float* cols = (float*)(at + b.cols_at);
    if (b.pass) {
        DzPassArgs a{dy, b.dz ? ws : nullptr, d->M, d->N, b.cols.rows, make};
        a.dz.cols = b.parts ? cols : nullptr;
        if (const int rc = status(o.dz(a, b.cols.gx, b.cols.gy, s), "psfm_linear_bwd: dz launch")) return rc;
    }
    PairArgs pair{};
    if (b.dx) {
        GemmArgs& a = pair.dx;
        a.P = dz, a.Q = w, a.ldp = d->N, a.ldq = d->K, a.I = d->M, a.J = d->K, a.R = d->N;
        a.e.out = dx, a.e.alpha = drop.scale, a.dz = make;
        set(a, b.pdx, at + b.dxp_at);
    }
    if (b.dw) {
        GemmArgs& a = pair.dw;
        a.P = dz, a.Q = x, a.ldp = d->N, a.ldq = d->ldx, a.I = d->N, a.J = d->K, a.R = d->M;
        a.e.out = dw, a.e.alpha = drop.scale, a.dz = make;
        if (db && !b.pass) (b.parts ? (void*&)a.dz.cols : a.dz.db) = b.parts ? (void*)cols : db;
        set(a, b.pdw, at + b.dwp_at);
    }
    const bool one = b.dx && b.dw && b.pdx.variant == b.pdw.variant &&
                     b.pdx.blocks() + b.pdw.blocks() <= most_blocks(LINEAR_TILES[b.pdx.variant].threads);
    for (int part = 0; part < (one ? 1 : 2); ++part) {
        pair.ndx = b.dx && part == 0 ? pair.dx.blocks() : 0;
        pair.ndw = b.dw && (one || part == 1) ? pair.dw.blocks() : 0;
        if (pair.ndx + pair.ndw == 0) continue;
        const int rc = o.pair(pair.ndx ? b.pdx.variant : b.pdw.variant, vec, b.stage, pair, s);
        if (rc) return status(rc, "psfm_linear_bwd: launch");
    }
    FinishArgs f{};
    f.dx = pair.dx, f.dw = pair.dw;
    // no rows or no products to sum: the bias gradient of no parts is zero
    if (db && d->N > 0 && (b.parts || !any)) f.cols = cols, f.parts = b.parts, f.N = d->N, f.alpha = drop.scale, f.db = db;
    return status(o.finish(f, s), "psfm_linear_bwd: finish launch");
}

const char* psfm_linear_last_error(void) { return g_err.c_str(); }

}  // extern "C"
