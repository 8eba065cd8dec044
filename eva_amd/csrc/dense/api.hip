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

// Parts of a sum of `k_tiles` for a result of `tiles` tiles of 128 by 128, so that a GPU's worth of workgroups runs: each adds its
// partial sums' way through memory, so it takes at least `least` k-tiles.
static int splits_of(int64_t tiles, int k_tiles, int least)
{
    if (tiles >= CUS || tiles == 0) return 1;
    int64_t n = (2 * CUS + tiles - 1) / tiles;
    if (n > k_tiles / least) n = k_tiles / least;
    if (n > MAX_SPLITS) n = MAX_SPLITS;
    return n < 1 ? 1 : (int)n;
}

static bool few_rows(int rows, int experts, bool grouped) { return grouped ? rows <= 32 * experts : rows <= 64; }

static int forward_splits(int rows, int k, int n, bool grouped)
{
    return grouped ? 1 : splits_of((int64_t)ceil_div(rows, 128) * ceil_div(n, 128), ceil_div(k, TILE_K), 4);
}
static size_t forward_part(int rows, int k, int n, bool grouped)
{
    const int s = forward_splits(rows, k, n, grouped);
    return s > 1 ? align256((size_t)s * rows * n * 4) : 0;
}
static int weight_splits(int rows, int n_in, int n_out, bool grouped)
{
    return grouped ? 1 : splits_of((int64_t)ceil_div(n_in, 128) * ceil_div(n_out, 128), ceil_div(rows, TILE_K), 4);
}
static size_t weight_part(int rows, int n_in, int n_out, bool grouped)
{
    const int s = weight_splits(rows, n_in, n_out, grouped);
    return s > 1 ? align256((size_t)s * n_in * n_out * 4) : 0;
}
static int column_parts(int rows, int n_out, int experts)
{
    const int64_t groups = (int64_t)ceil_div(n_out, 512) * experts;
    int64_t n = (4 * CUS + groups - 1) / groups;
    if (n > rows / 32) n = rows / 32;
    if (n > 64) n = 64;
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

// Rows that the direct loads take: 16-byte addresses and lengths, 32-bit offsets.
static bool direct(const void* p, int64_t stride, int64_t rows, int len)
{
    return (((uintptr_t)p | (uintptr_t)(2 * stride)) & 15) == 0 && len % 8 == 0 && (rows + 512) * stride * 2 < 0xf0000000ll;
}

}  // namespace evamx_dense

using namespace evamx_dense;

extern "C" const char* evamx_dense_last_error(void) { return g_error; }
extern "C" int evamx_dense_version(void) { return EVAMX_DENSE_VERSION; }

extern "C" size_t evamx_linear_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped)
{
    set_error("%s", "");
    if (!sizes_ok("evamx_linear_workspace_bytes", rows, n_in, n_out, experts, grouped)) return 0;
    return few_rows(rows, experts, grouped) ? 0 : forward_part(rows, n_in, n_out, grouped);
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
    const size_t need = evamx_linear_workspace_bytes(a->rows, a->n_in, a->n_out, a->experts, grouped);
    if (!space_ok(who, a->workspace, a->workspace_bytes, need)) return need > a->workspace_bytes && a->workspace ? EVAMX_ENOSPACE : EVAMX_EINVAL;
    LinearParams p = {};
    p.x = (const uint16_t*)a->x; p.w = (const uint16_t*)a->w; p.bias = (const uint16_t*)a->bias; p.residual = (const uint16_t*)a->residual;
    p.y = (uint16_t*)a->y; p.pre = a->pre;
    p.x_stride = (size_t)a->x_stride; p.w_stride = (size_t)a->w_stride; p.w_expert_stride = (size_t)a->w_expert_stride;
    p.residual_stride = (size_t)a->residual_stride; p.y_stride = (size_t)a->y_stride;
    p.g = Groups{a->starts, a->experts, a->rows};
    p.n_in = a->n_in; p.n_out = a->n_out; p.inter = a->act == EVAMX_ACT_SWIGLU ? cols : 0;
    p.act = a->act; p.limit = a->limit;
    p.splits = 1;
    const bool loose = !direct(a->x, a->x_stride, 256, a->n_in) || !direct(a->w, a->w_stride, a->n_out, a->n_in) ||
                       (a->experts > 1 && a->w_expert_stride % 8);
    if (few_rows(a->rows, a->experts, grouped)) return launch_few(p, a->dtype, loose, (hipStream_t)stream);
    p.splits = forward_splits(a->rows, a->n_in, a->n_out, grouped);
    p.part = (float*)a->workspace;
    return launch_tiles(p, a->dtype, false, loose, (hipStream_t)stream);
}

extern "C" size_t evamx_linear_grad_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped, int act)
{
    set_error("%s", "");
    if (!sizes_ok("evamx_linear_grad_workspace_bytes", rows, n_in, n_out, experts, grouped)) return 0;
    size_t part = forward_part(rows, n_out, n_in, grouped);
    const size_t w = weight_part(rows, n_in, n_out, grouped), c = column_part(rows, n_out, experts);
    if (w > part) part = w;
    if (c > part) part = c;
    return part + (act != EVAMX_ACT_NONE ? align256((size_t)rows * ((n_out + 7) / 8 * 8) * 2) : 0);
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
    const size_t need = evamx_linear_grad_workspace_bytes(a->rows, a->n_in, a->n_out, a->experts, grouped, a->act);
    if (!space_ok(who, a->workspace, a->workspace_bytes, need)) return need > a->workspace_bytes && a->workspace ? EVAMX_ENOSPACE : EVAMX_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    const Groups g{a->starts, a->experts, a->rows};
    const uint16_t* d = (const uint16_t*)a->grad;
    size_t d_stride = (size_t)a->grad_stride;
    char* ws = (char*)a->workspace;
    if (a->act != EVAMX_ACT_NONE) {
        d_stride = (size_t)(a->n_out + 7) / 8 * 8;
        uint16_t* out = (uint16_t*)ws;
        ws += align256((size_t)a->rows * d_stride * 2);
        d = out;
        if (a->rows) {
            const int rc = launch_act_grad(ActGradParams{(const uint16_t*)a->grad, (size_t)a->grad_stride, a->pre, out, d_stride, g, a->n_out,
                                                         a->act, a->limit}, a->dtype, s);
            if (rc != EVAMX_OK) return rc;
        }
    }
    const bool loose_d = !direct(d, (int64_t)d_stride, 256, a->n_out);
    if (a->grad_x && a->rows) {
        LinearParams p = {};
        p.x = d; p.x_stride = d_stride; p.w = (const uint16_t*)a->w; p.w_stride = (size_t)a->w_stride; p.w_expert_stride = (size_t)a->w_expert_stride;
        p.y = (uint16_t*)a->grad_x; p.y_stride = (size_t)a->grad_x_stride;
        p.g = g; p.n_in = a->n_out; p.n_out = a->n_in;
        p.splits = forward_splits(a->rows, a->n_out, a->n_in, grouped);
        p.part = (float*)ws;
        const bool loose = loose_d || !direct(a->w, a->w_stride, TILE_K, a->n_in) || (a->experts > 1 && a->w_expert_stride % 8);
        const int rc = launch_tiles(p, a->dtype, true, loose, s);
        if (rc != EVAMX_OK) return rc;
    }
    if (a->grad_w) {
        WeightGradParams p = {(const uint16_t*)a->x, d, (size_t)a->x_stride, d_stride, (uint16_t*)a->grad_w, g, a->n_in, a->n_out, (float*)ws,
                              weight_splits(a->rows, a->n_in, a->n_out, grouped)};
        const int rc = launch_weight_grad(p, a->dtype, loose_d || !direct(a->x, a->x_stride, TILE_K, a->n_in), s);
        if (rc != EVAMX_OK) return rc;
    }
    if (a->grad_bias) {
        ColumnSumParams p = {d, d_stride, (uint16_t*)a->grad_bias, g, a->n_out, (float*)ws, column_parts(a->rows, a->n_out, a->experts)};
        return launch_column_sums(p, a->dtype, s);
    }
    return EVAMX_OK;
}
