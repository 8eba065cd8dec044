// The entry points: checks, the choice of kernels, the workspace.
#include <stdarg.h>
#include <stdio.h>

#include "grads.hpp"

namespace evamx_dense {

static thread_local char g_error[512];

void set_error(const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

int launched(const char* what)
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return EVAMX_OK;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return EVAMX_ELAUNCH;
}

constexpr int MAX_ROWS = 1 << 24, MAX_SPLITS = 16;

static size_t align256(size_t n) { return (n + 255) / 256 * 256; }

static Plan plan_with(int64_t rows, int64_t cols, int64_t k, double& least)
{
    const int64_t kt = (k + TILE_K - 1) / TILE_K;
    Plan best = {TILES_256, 1};
    least = 1e30;
    for (int size : {TILES_128, TILES_256})
        for (int splits = 1; splits <= MAX_SPLITS && (splits == 1 || kt / splits >= 4); ++splits) {
            const int64_t edge = size == TILES_256 ? 256 : 128, at_once = size == TILES_256 ? CUS : 2 * CUS;
            const int64_t work = ((rows + edge - 1) / edge) * ((cols + edge - 1) / edge) * splits, rest = work % at_once;
            const double each = (double)((kt + splits - 1) / splits);
            auto round = [&](int64_t n) {
                if (size == TILES_256) return each * (1.15 + (n > 160 ? 0.35 * (n - 160) / (CUS - 160) : 0)) + 5;
                return each * (n <= CUS ? 0.58 + 0.04 * n / CUS : 0.62 + 0.23 * (n - CUS) / CUS) + 4;
            };
            double time = (double)(work / at_once) * round(at_once) + (rest ? round(rest) : 0);
            // what is read, at the rate that so many workgroups reach
            const double many = (double)work / (size == TILES_256 ? 210 : 430), few = size == TILES_256 ? 0.2 : 0.4;
            const double read = 2.0 * (rows + cols) * k / (4.9e6 * (few + (1 - few) * (many < 1 ? many : 1)));
            if (time < read) time = read;
            if (splits > 1) time += 7 + (double)splits * rows * cols * 4 / 2.9e6;
            if (time < least) {
                least = time;
                best = {size, splits};
            }
        }
    return best;
}

Plan plan_of(int64_t rows, int64_t cols, int64_t k)
{
    double least;
    return plan_with(rows, cols, k, least);
}

// Whether few.hip takes a call: for one matrix where its time (6 us, the weights at 5.6 TB/s, and the rows of x, which each workgroup
// reads, at 8.9) is below the tiles', up to 64 rows (measured, us, at 1, 16 and 64 rows: 7168 -> 2048: 12, 16, 35 against 19, 20, 21;
// 7168 -> 18432: 51, 82, 188 against 56, 56, 62). For experts up to four rows for each, of which most may be another rank's, whatever
// the experts' shares (64 experts, 7168 -> 4096, rows for four each: spread evenly 544 against 664, by Zipf's law 605 against 633, all
// one expert's 84 against 134), but not for many workgroups that have little to sum (64 experts, 512 -> 1024: 33 against 18; 32, 1024
// -> 768: 16 against 20), unless tiles had to copy the weights (24, 333 -> 1000: 16 against 26).
static bool few_rows(int rows, int k, int n, int experts, bool grouped, bool direct)
{
    if (grouped) return rows <= 4 * (int64_t)experts && (k >= 1024 || ceil_div(n, 16) * (int64_t)experts <= 1024 || !direct);
    if (rows > 64) return false;
    double tiles;
    plan_with(rows, n, k, tiles);
    const double x = ceil_div(n, rows > 8 && n >= 24 * CUS ? 32 : 16) * (double)rows * k * 2;
    return 6 + (double)n * k * 2 / 5.6e6 + x / 8.9e6 <= tiles;
}

// More rows than that may still be few of each expert, or most of them other ranks': where the weights are more than the caches hold, few.hip
// takes the experts of up to 16 rows and the tiles the others (64 experts, 7168 -> 4096, 8 rows each: 568 us against 667 with tiles
// alone, 16: 635 against 675; a rank's eighth of 32 rows each: 551 against 665; by Zipf's law 32 rows for each: 766 against 876). Where
// no expert has as few, the launch without work costs 8 to 22 (60 rows each: 708 against 695; 2048 -> 7168: 405 against 383).
constexpr int FEW_OF_MANY = 16, MANY = 64;

// Experts' rows are known to the device alone: large tiles (which the kernel takes by halves and quarters where an expert ends), if
// the most there can be fill the GPU.
static Plan forward_plan(int rows, int k, int n, int experts, bool grouped)
{
    if (!grouped) return plan_of(rows, n, k);
    return {(rows / 256 + (rows < experts ? rows : experts)) * (int64_t)ceil_div(n, 256) >= CUS * 3 / 4 ? TILES_256 : TILES_128, 1};
}
static size_t forward_part(int rows, int k, int n, int experts, bool grouped)
{
    const int s = forward_plan(rows, k, n, experts, grouped).splits;
    return s > 1 ? align256((size_t)s * rows * n * 4) : 0;
}
static Plan weight_plan(int rows, int n_in, int n_out, int experts, bool grouped)
{
    if (!grouped) return plan_of(n_out, n_in, rows);
    return {(int64_t)ceil_div(n_out, 256) * ceil_div(n_in, 256) * experts >= CUS * 3 / 4 ? TILES_256 : TILES_128, 1};
}
static size_t weight_part(int rows, int n_in, int n_out, int experts, bool grouped)
{
    const int s = weight_plan(rows, n_in, n_out, experts, grouped).splits;
    return s > 1 ? align256((size_t)s * n_in * n_out * 4) : 0;
}
// Runs of rows whose column sums are made apart: enough for the GPU, at least 32 rows each.
static int column_parts(int rows, int n_out, int experts)
{
    const int64_t groups = (int64_t)ceil_div(n_out, 512) * experts;
    int64_t n = (CUS + groups - 1) / groups;
    if (n > rows / 32) n = rows / 32;
    if (n > 32) n = 32;
    return n < 1 ? 1 : (int)n;
}
static size_t column_part(int rows, int n_out, int experts)
{
    const int n = column_parts(rows, n_out, experts);
    return n > 1 ? align256((size_t)n * experts * n_out * 4) : 0;
}

static bool sizes_ok(const char* who, int rows, int n_in, int n_out, int experts, bool grouped)
{
    if (rows < 0 || rows > MAX_ROWS) { set_error("%s: rows %d outside 0..%d", who, rows, MAX_ROWS); return false; }
    if (n_in < 1 || n_in > EVAMX_W4_MAX_DIM || n_out < 1 || n_out > EVAMX_W4_MAX_DIM) {
        set_error("%s: a matrix of %d by %d (1..%d)", who, n_out, n_in, EVAMX_W4_MAX_DIM);
        return false;
    }
    if (experts < 1 || experts > MAX_EXPERTS || (!grouped && experts != 1)) {
        set_error("%s: %d experts (1..%d; 1 without starts)", who, experts, MAX_EXPERTS);
        return false;
    }
    return true;
}

static bool act_ok(const char* who, int act, float limit, int n_out)
{
    if (act < EVAMX_ACT_NONE || act > EVAMX_ACT_SWIGLU) { set_error("%s: activation %d", who, act); return false; }
    if (act == EVAMX_ACT_SWIGLU && n_out % 2) { set_error("%s: SwiGLU of %d columns", who, n_out); return false; }
    if (!(limit >= 0) || (limit != 0 && act != EVAMX_ACT_SWIGLU)) { set_error("%s: limit %g (SwiGLU's, 0 or more)", who, limit); return false; }
    return true;
}

static bool space_ok(const char* who, const void* ws, size_t have, size_t need)
{
    if (need == 0) return true;
    if (!ws || ((uintptr_t)ws & 15)) { set_error("%s: the workspace must be 16-byte aligned", who); return false; }
    if (have < need) { set_error("%s: workspace %zu bytes < %zu", who, have, need); return false; }
    return true;
}

// Rows that tiles take as they are: 16-byte addresses and lengths, and strides whose multiples in a tile stay 32-bit offsets.
static bool direct(const void* p, int64_t stride, int len)
{
    return (((uintptr_t)p | (uintptr_t)(2 * stride)) & 15) == 0 && len % 8 == 0 && stride <= 1 << 21;
}

static int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
static size_t padded(int64_t rows, int n) { return align256((size_t)rows * pad8(n) * 2); }

// Rows that tiles take: as they are, or copied to `at`, which moves on.
struct Rows {
    const uint16_t* p;
    int64_t stride, matrix_stride;
};
static int ready(Rows& r, bool as_is, int64_t rows, int count, int n, char*& at, hipStream_t s)
{
    if (as_is) return EVAMX_OK;
    uint16_t* to = (uint16_t*)at;
    at += padded(rows * count, n);
    const int rc = launch_pad(r.p, (size_t)r.stride, (size_t)r.matrix_stride, (int)rows, count, n, to, s);
    r = Rows{to, pad8(n), rows * pad8(n)};
    return rc;
}
static int lie_of(const void* p, int64_t stride, int64_t matrix_stride)
{
    const uint64_t all = (uint64_t)(uintptr_t)p | (uint64_t)(2 * stride) | (uint64_t)(2 * matrix_stride);
    return all & 3 ? LIE_2 : all & 15 ? LIE_4 : LIE_16;
}

}  // namespace evamx_dense

using namespace evamx_dense;

extern "C" const char* evamx_dense_last_error(void) { return g_error; }
extern "C" int evamx_dense_version(void) { return EVAMX_DENSE_VERSION; }

// What a call may copy of x and w: both, unless their sizes rule it out (their addresses and strides are the call's).
static size_t forward_copies(int rows, int n_in, int n_out, int experts) { return padded(rows, n_in) + padded((int64_t)n_out * experts, n_in); }

extern "C" size_t evamx_linear_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped, int direct)
{
    set_error("%s", "");
    if (!sizes_ok("evamx_linear_workspace_bytes", rows, n_in, n_out, experts, grouped)) return 0;
    if (few_rows(rows, n_in, n_out, experts, grouped, direct)) return 0;
    return forward_part(rows, n_in, n_out, experts, grouped) + (direct ? 0 : forward_copies(rows, n_in, n_out, experts));
}

// Whether a forward call takes x and w as they are.
static bool x_direct(const evamx_linear_args* a) { return direct(a->x, a->x_stride, a->n_in); }
static bool w_direct(const void* w, int64_t stride, int64_t matrix, int experts, int n_in)
{
    return direct(w, stride, n_in) && (experts == 1 || matrix % 8 == 0);
}

extern "C" int evamx_linear(const evamx_linear_args* a, evamx_stream_t stream)
{
    const char* who = "evamx_linear";
    set_error("%s", "");
    if (!a) { set_error("%s: null arguments", who); return EVAMX_EINVAL; }
    const bool grouped = a->starts != nullptr;
    if (!sizes_ok(who, a->rows, a->n_in, a->n_out, a->experts, grouped) || !act_ok(who, a->act, a->limit, a->n_out)) return EVAMX_EINVAL;
    if (a->dtype != EVAMX_DTYPE_F16 && a->dtype != EVAMX_DTYPE_BF16) { set_error("%s: dtype %d", who, a->dtype); return EVAMX_EINVAL; }
    const int cols = a->act == EVAMX_ACT_SWIGLU ? a->n_out / 2 : a->n_out;
    if (a->x_stride < a->n_in || a->w_stride < a->n_in || a->y_stride < cols || (a->residual && a->residual_stride < cols) ||
        (a->experts > 1 && a->w_expert_stride < a->w_stride * (int64_t)(a->n_out - 1) + a->n_in)) {
        set_error("%s: strides below the row lengths", who);
        return EVAMX_EINVAL;
    }
    if (a->rows == 0) return EVAMX_OK;
    if (!a->x || !a->w || !a->y) { set_error("%s: null pointer", who); return EVAMX_EINVAL; }
    const bool xd = x_direct(a), wd = w_direct(a->w, a->w_stride, a->w_expert_stride, a->experts, a->n_in);
    const size_t need = evamx_linear_workspace_bytes(a->rows, a->n_in, a->n_out, a->experts, grouped, xd && wd);
    if (!space_ok(who, a->workspace, a->workspace_bytes, need)) return need > a->workspace_bytes && a->workspace ? EVAMX_ENOSPACE : EVAMX_EINVAL;
    LinearParams p = {};
    Rows x = {(const uint16_t*)a->x, a->x_stride, 0}, w = {(const uint16_t*)a->w, a->w_stride, a->experts > 1 ? a->w_expert_stride : 0};
    p.bias = (const uint16_t*)a->bias; p.residual = (const uint16_t*)a->residual;
    p.y = (uint16_t*)a->y; p.pre = a->pre;
    p.residual_stride = (size_t)a->residual_stride; p.y_stride = (size_t)a->y_stride;
    p.g = Groups{a->starts, a->experts, a->rows};
    p.n_in = a->n_in; p.n_out = a->n_out; p.inter = a->act == EVAMX_ACT_SWIGLU ? cols : 0;
    p.act = a->act; p.limit = a->limit;
    p.splits = 1; p.stream = (int64_t)a->rows * cols * 2 > CACHE;
    const hipStream_t s = (hipStream_t)stream;
    const bool few = few_rows(a->rows, a->n_in, a->n_out, a->experts, grouped, xd && wd);
    if (!few) {
        char* at = (char*)a->workspace;
        int rc = ready(x, xd, a->rows, 1, a->n_in, at, s);
        if (rc == EVAMX_OK) rc = ready(w, wd, a->n_out, a->experts, a->n_in, at, s);
        if (rc != EVAMX_OK) return rc;
        const Plan plan = forward_plan(a->rows, a->n_in, a->n_out, a->experts, grouped);
        p.size = plan.size; p.splits = plan.splits; p.part = (float*)at;
        p.x_cols = p.w_cols = (int)pad8(a->n_in);
        if (p.inter && (a->n_out + 512) * w.stride * 2 >= 0xf0000000ll) {    // one descriptor spans the gate's and the up product's rows
            set_error("%s: a SwiGLU matrix of %d rows %lld apart", who, a->n_out, (long long)w.stride);
            return EVAMX_EINVAL;
        }
    }
    p.x = x.p; p.x_stride = (size_t)x.stride; p.w = w.p; p.w_stride = (size_t)w.stride; p.w_expert_stride = (size_t)w.matrix_stride;
    const bool large = (int64_t)a->experts * a->n_out * a->n_in * 2 > CACHE;
    if (!few) {
        if (grouped && large && xd && wd && a->rows <= MANY * (int64_t)a->experts) {
            p.g.upto = FEW_OF_MANY;
            const int rc = launch_few(p, a->dtype, LIE_STREAM, s);
            if (rc != EVAMX_OK) return rc;
            p.g.above = FEW_OF_MANY; p.g.upto = Groups::ALL;
        }
        return launch_tiles(p, a->dtype, false, s);
    }
    const int lx = lie_of(a->x, a->x_stride, 0), lw = lie_of(a->w, a->w_stride, a->experts > 1 ? a->w_expert_stride : 0);
    int lie = lx > lw ? lx : lw;
    if (lie == LIE_16 && a->n_in % 8) lie = LIE_4;
    if (lie == LIE_16 && large) lie = LIE_STREAM;
    return launch_few(p, a->dtype, lie, s);
}

// What a gradient call may copy: D (where there is no activation to write it anew), x and w.
static size_t grad_copies(int rows, int n_in, int n_out, int experts)
{
    return padded(rows, n_out) + padded(rows, n_in) + padded((int64_t)n_out * experts, n_in);
}

extern "C" size_t evamx_linear_grad_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped, int act, int direct)
{
    set_error("%s", "");
    if (!sizes_ok("evamx_linear_grad_workspace_bytes", rows, n_in, n_out, experts, grouped)) return 0;
    size_t part = forward_part(rows, n_out, n_in, experts, grouped);
    const size_t w = weight_part(rows, n_in, n_out, experts, grouped), c = column_part(rows, n_out, experts);
    if (w > part) part = w;
    if (c > part) part = c;
    return part + (direct ? act != EVAMX_ACT_NONE ? padded(rows, n_out) : 0 : grad_copies(rows, n_in, n_out, experts));
}

extern "C" int evamx_linear_grad(const evamx_linear_grad_args* a, evamx_stream_t stream)
{
    const char* who = "evamx_linear_grad";
    set_error("%s", "");
    if (!a) { set_error("%s: null arguments", who); return EVAMX_EINVAL; }
    const bool grouped = a->starts != nullptr;
    if (!sizes_ok(who, a->rows, a->n_in, a->n_out, a->experts, grouped) || !act_ok(who, a->act, a->limit, a->n_out)) return EVAMX_EINVAL;
    if (a->dtype != EVAMX_DTYPE_F16 && a->dtype != EVAMX_DTYPE_BF16) { set_error("%s: dtype %d", who, a->dtype); return EVAMX_EINVAL; }
    const int cols = a->act == EVAMX_ACT_SWIGLU ? a->n_out / 2 : a->n_out;
    if (a->grad_stride < cols || (a->grad_w && a->x_stride < a->n_in) || (a->grad_x && (a->w_stride < a->n_in || a->grad_x_stride < a->n_in)) ||
        (a->grad_x && a->experts > 1 && a->w_expert_stride < a->w_stride * (int64_t)(a->n_out - 1) + a->n_in)) {
        set_error("%s: strides below the row lengths", who);
        return EVAMX_EINVAL;
    }
    if (a->rows && (!a->grad || (a->grad_w && !a->x) || (a->grad_x && !a->w) || (a->act != EVAMX_ACT_NONE && !a->pre))) {
        set_error("%s: null pointer", who);
        return EVAMX_EINVAL;
    }
    const bool act = a->act != EVAMX_ACT_NONE;
    const bool dd = act || direct(a->grad, a->grad_stride, a->n_out), xd = direct(a->x, a->x_stride, a->n_in);
    const bool wd = w_direct(a->w, a->w_stride, a->w_expert_stride, a->experts, a->n_in);
    const bool all = dd && (!a->grad_w || xd) && (!a->grad_x || wd);
    const size_t need = evamx_linear_grad_workspace_bytes(a->rows, a->n_in, a->n_out, a->experts, grouped, a->act, all);
    if (!space_ok(who, a->workspace, a->workspace_bytes, need)) return need > a->workspace_bytes && a->workspace ? EVAMX_ENOSPACE : EVAMX_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    const Groups g{a->starts, a->experts, a->rows};
    char* at = (char*)a->workspace;
    Rows d = {(const uint16_t*)a->grad, a->grad_stride, 0}, x = {(const uint16_t*)a->x, a->x_stride, 0};
    Rows w = {(const uint16_t*)a->w, a->w_stride, a->experts > 1 ? a->w_expert_stride : 0};
    int rc = EVAMX_OK;
    if (act) {
        uint16_t* out = (uint16_t*)at;
        at += padded(a->rows, a->n_out);
        d = Rows{out, pad8(a->n_out), 0};
        if (a->rows)
            rc = launch_act_grad(ActGradParams{(const uint16_t*)a->grad, (size_t)a->grad_stride, a->pre, out, (size_t)d.stride, g, a->n_out, a->act,
                                               a->limit}, a->dtype, s);
    } else if (a->rows && (a->grad_x || a->grad_w)) {
        rc = ready(d, dd, a->rows, 1, a->n_out, at, s);
    }
    if (rc == EVAMX_OK && a->grad_w && a->rows) rc = ready(x, xd, a->rows, 1, a->n_in, at, s);
    if (rc == EVAMX_OK && a->grad_x && a->rows) rc = ready(w, wd, a->n_out, a->experts, a->n_in, at, s);
    if (rc != EVAMX_OK) return rc;
    if (a->grad_x && a->rows) {
        LinearParams p = {};
        p.x = d.p; p.x_stride = (size_t)d.stride; p.w = w.p; p.w_stride = (size_t)w.stride; p.w_expert_stride = (size_t)w.matrix_stride;
        p.y = (uint16_t*)a->grad_x; p.y_stride = (size_t)a->grad_x_stride;
        p.g = g; p.n_in = a->n_out; p.n_out = a->n_in; p.x_cols = (int)pad8(a->n_out); p.w_cols = (int)pad8(a->n_in);
        const Plan plan = forward_plan(a->rows, a->n_out, a->n_in, a->experts, grouped);
        p.size = plan.size; p.splits = plan.splits; p.part = (float*)at; p.stream = (int64_t)a->rows * a->n_in * 2 > CACHE;
        rc = launch_tiles(p, a->dtype, true, s);
        if (rc != EVAMX_OK) return rc;
    }
    if (a->grad_w) {
        WeightGradParams p = {x.p, d.p, (size_t)x.stride, (size_t)d.stride, (uint16_t*)a->grad_w, g,
                              (int64_t)a->experts * a->n_in * a->n_out * 2 > CACHE, a->n_in, a->n_out, (int)pad8(a->n_in),
                              (int)pad8(a->n_out), (float*)at, weight_plan(a->rows, a->n_in, a->n_out, a->experts, grouped)};
        rc = launch_weight_grad(p, a->dtype, s);
        if (rc != EVAMX_OK) return rc;
    }
    if (a->grad_bias) {
        ColumnSumParams p = {d.p, (size_t)d.stride, (uint16_t*)a->grad_bias, g, a->n_out, (float*)at, column_parts(a->rows, a->n_out, a->experts)};
        return launch_column_sums(p, a->dtype, s);
    }
    return EVAMX_OK;
}
