// y = x W^T (+ bias) on 4-bit weights with group scales (w4.hpp).
#include "evamx_gemv.hpp"
#include "evamx_internal.hpp"
#include "w4_gemm.hpp"

namespace evamx {

struct W4LinearParams {
    const void* x;               // as given
    size_t x_stride;
    const w4_half* xh;           // made ready: rows of kt * 128
    const float* row_scale;      // NULL: 1
    int rows, aligned, y_aligned, bf16;          // x's and y's rows start at 16-byte addresses
    const void* bias;
    void* y;
    size_t y_stride;
};

__device__ __forceinline__ float w4_bias(const void* b, int n, int bf16)
{
    return bf16 ? __builtin_bit_cast(float, (uint32_t)((const uint16_t*)b)[n] << 16) : (float)((const w4_half*)b)[n];
}

__device__ __forceinline__ void w4_linear_store(const W4LinearParams& p, const W4Mat& m, int row, int n, float v, float scale)
{
    v *= scale;
    if (p.bias) v += w4_bias(p.bias, n, p.bf16);
    w4_store(p.y, (size_t)row * p.y_stride + n, v, p.bf16);
}

// Up to four rows: one launch. A workgroup takes 16 columns, a wave one part of the k-tiles; the rows are made ready in LDS
// while the first tiles are on their way, and each stands in four of the 16 rows of a matrix operand, so that one of the four
// accumulators of a lane is all there is to scale. 2048 -> 7168 at one row: 4.9 us in a graph, of which an empty launch is 1.6;
// the rest is the loads' one round trip and the join.
template <int SG, bool ZERO>
__global__ __launch_bounds__(512) void w4_linear_few_kernel(W4LinearParams p, W4Mat m)
{
    extern __shared__ w4_half xs[];
    __shared__ uint32_t top[W4_MAX_PARTS][4];
    __shared__ float scale[4], part[W4_MAX_PARTS][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, parts = blockDim.x >> 6, ld = m.kt * W4_TILE_K + W4_STAGE_PAD;
    const int k0 = w4_part_begin(m.kt, parts, wave), k1 = w4_part_begin(m.kt, parts, wave + 1);
    W4Stage stage{(const uint16_t*)p.x, p.x_stride, p.rows, m.n_in, m.kt, p.bf16, p.aligned};
    stage.load();
    const W4Stream st[1] = {w4_stream<SG, ZERO>(m, 0, blockIdx.x, k1)};
    const int row = (lane & 15) >> 2;
    const w4_half* a = xs + (row < p.rows ? row : p.rows - 1) * ld + 8 * (lane >> 4);
    w4_f32x4 acc[1][1] = {};
    w4_run<2, SG, ZERO, 1, 1, 1, false>(
        acc, st, k0, k1, m.bf16, [](int, int) {},
        [&](int, int kt, w4_half8 (&x)[1][4], w4_half8 (&)[1][4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[0][j] = *(const w4_half8*)(a + kt * W4_TILE_K + 32 * j);
        },
        [&] { stage.finish(xs, top, scale); });
    part[wave][lane] = acc[0][0][0];
    __syncthreads();
    if (wave) return;
    const int r = lane >> 4, n = 16 * blockIdx.x + (lane & 15);
    if (r >= p.rows || n >= m.n_out) return;
    float v = 0;
    for (int w = 0; w < parts; ++w) v += part[w][lane];
    w4_linear_store(p, m, r, n, v, scale[r]);
}

// 16 MB rows by 16 NB columns a workgroup, a wave one part of the k-tiles; the rows come ready from memory (L2) with the tiles.
// 7168 -> 18432 with groups of 64 and zero points at 5 rows: 19.6 us, 3.7 TB/s; 7168 -> 2048 at 200 rows: 21.5 us, 273 TFLOP/s,
// bound by the rows' operands, 8 KiB a k-tile and wave beside 4 of codes, which no wave shares with another.
template <int SG, bool ZERO, int NB, int MB>
__global__ __launch_bounds__(512) void w4_linear_kernel(W4LinearParams p, W4Mat m)
{
    extern __shared__ w4_f32x4 part[];                       // [parts][NB][MB][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, parts = blockDim.x >> 6;
    const int k0 = w4_part_begin(m.kt, parts, wave), k1 = w4_part_begin(m.kt, parts, wave + 1), r0 = 16 * MB * blockIdx.y;
    W4Stream st[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int nt = NB * blockIdx.x + b;
        st[b] = w4_stream<SG, ZERO>(m, 0, nt < m.nt ? nt : m.nt - 1, k1);
    }
    W4GlobalRows<MB, false> rows;
    rows.src = w4_rsrc(p.xh + (size_t)r0 * m.kt * W4_TILE_K, (uint32_t)(p.rows - r0 < 16 * MB ? p.rows - r0 : 16 * MB) * m.kt * (W4_TILE_K * 2));
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int r = 16 * mb + (lane & 15);
        rows.at[mb] = (uint32_t)(r0 + r < p.rows ? r : p.rows - 1 - r0) * m.kt * (W4_TILE_K * 2) + 16 * (lane >> 4);
    }
    w4_f32x4 acc[NB][MB] = {};
    w4_run<1, SG, ZERO, NB, MB, 4, false>(
        acc, st, k0, k1, m.bf16, [&](int, int kt) { rows.request(kt); },
        [&](int, int, w4_half8 (&x)[MB][4], w4_half8 (&lo)[MB][4]) { rows.take(x, lo); }, [] {});
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) part[((wave * NB + b) * MB + mb) * 64 + lane] = acc[b][mb];
    __syncthreads();
    for (int t = wave; t < NB * MB * 4; t += parts) {        // value i of block mb and stream b
        const int i = t & 3, mb = (t >> 2) % MB, b = (t >> 2) / MB;
        const int r = r0 + 16 * mb + 4 * (lane >> 4) + i, n = 16 * (NB * blockIdx.x + b) + (lane & 15);
        if (r >= p.rows || n >= m.n_out) continue;
        float v = 0;
        for (int w = 0; w < parts; ++w) v += part[((w * NB + b) * MB + mb) * 64 + lane][i];
        w4_linear_store(p, m, r, n, v, p.row_scale ? p.row_scale[r] : 1.0f);
    }
}

// Long calls: 64 rows by 256 columns a workgroup (w4_gemm.hpp). Consecutive workgroups go to the eight XCDs in turn, so each XCD
// takes a contiguous run of tiles, eight row tiles by all columns at a time: its rows' tiles stay in its L2 while it passes over
// the columns. 8192 rows of 2048 -> 7168: about 225 us, 1070 TFLOP/s, in a graph (242 and more in a trace), and 13 to make the bf16
// rows ready.
template <int SG, bool ZERO, int MB>
__device__ __forceinline__ void w4_linear_gemm(const W4LinearParams& p, const W4Mat& m, int r0, int have, int nt0, char* lds)
{
    W4Stream st[W4G_NB];
#pragma unroll
    for (int b = 0; b < W4G_NB; ++b) st[b] = w4_stream<SG, ZERO>(m, 0, nt0 + b < m.nt ? nt0 + b : m.nt - 1, m.kt);
    W4GemmRows<MB> rows;
    const uint32_t ld = m.kt * (W4_TILE_K * 2);
    rows.src = w4_rsrc(p.xh + (size_t)r0 * m.kt * W4_TILE_K, have * ld);
#pragma unroll
    for (int i = 0; i < MB; ++i) rows.at[i] = (w4g_row<MB>(i) < have ? w4g_row<MB>(i) : have - 1) * ld + w4g_chunk<MB>(i);
    w4_f32x4 acc[W4G_NB][MB] = {};
    w4g_run<SG, ZERO, false, MB>(acc, st, rows, lds, m.kt, m.bf16);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();                                         // no wave reads the rows' tiles any more
    if (16 * (nt0 + W4G_NB) <= m.n_out && p.y_aligned) {
        // whole columns: through LDS (a piece of its own a wave, rows 144 bytes apart: no two of a store's rows in the same banks)
        // into 16-byte pieces of the rows
        constexpr int ROW = 144;
        char* mine = lds + wave * (W4G_ROWS * ROW);
        float bias[W4G_NB];
#pragma unroll
        for (int b = 0; b < W4G_NB; ++b) bias[b] = p.bias ? w4_bias(p.bias, 16 * (nt0 + b) + (lane & 15), p.bf16) : 0.0f;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * mb + 4 * (lane >> 4) + i;
                const float f = p.row_scale ? p.row_scale[r0 + (r < have ? r : have - 1)] : 1.0f;
#pragma unroll
                for (int b = 0; b < W4G_NB; ++b)
                    *(uint16_t*)(mine + r * ROW + 2 * (16 * b + (lane & 15))) = w4_bits(p.bias ? acc[b][mb][i] * f + bias[b] : acc[b][mb][i] * f, p.bf16);
            }
        wave_lds_fence();
#pragma unroll
        for (int k = 0; k < 2 * MB; ++k) {
            const int r = 8 * k + (lane >> 3);
            if (r < have) *(w4_u32x4*)((uint16_t*)p.y + (size_t)(r0 + r) * p.y_stride + 16 * nt0 + 8 * (lane & 7)) = *(const w4_u32x4*)(mine + r * ROW + 16 * (lane & 7));
        }
        return;
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + 16 * mb + 4 * (lane >> 4) + i;
            if (r >= p.rows) continue;
            const float f = p.row_scale ? p.row_scale[r] : 1.0f;
#pragma unroll
            for (int b = 0; b < W4G_NB; ++b) {
                const int n = 16 * (nt0 + b) + (lane & 15);
                if (n < m.n_out) w4_linear_store(p, m, r, n, acc[b][mb][i], f);
            }
        }
}

template <int SG, bool ZERO>
__global__ __launch_bounds__(256, 2) void w4_linear_gemm_kernel(W4LinearParams p, W4Mat m, int row_tiles, int col_tiles)
{
    __shared__ __attribute__((aligned(128))) char lds[w4g_lds<false>()];
    const int total = row_tiles * col_tiles, per = w4_ceil(total, 8), t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || t >= total) return;
    const int band = t / (8 * col_tiles), in_band = t - band * 8 * col_tiles, deep = row_tiles - 8 * band < 8 ? row_tiles - 8 * band : 8;
    const int r0 = W4G_ROWS * (8 * band + in_band % deep), have = p.rows - r0 < W4G_ROWS ? p.rows - r0 : W4G_ROWS;
    const int nt0 = W4G_COLS / 16 * (in_band / deep) + (threadIdx.x >> 6) * W4G_NB;
    if (have > 32) w4_linear_gemm<SG, ZERO, 4>(p, m, r0, have, nt0, lds);
    else if (have > 16) w4_linear_gemm<SG, ZERO, 2>(p, m, r0, have, nt0, lds);
    else w4_linear_gemm<SG, ZERO, 1>(p, m, r0, have, nt0, lds);
}

constexpr int W4_CUS = 256;                                  // of an MI355X

template <int NB, int MB>
static void w4_launch_linear(const W4LinearParams& p, const W4Mat& m, const evamx_w4_weight& w, int parts, hipStream_t s)
{
    const dim3 grid(w4_ceil(m.nt, NB), w4_ceil(p.rows, 16 * MB));
    w4_dispatch(w, [&](auto sg, auto zero) {
        w4_linear_kernel<decltype(sg)::value, decltype(zero)::value, NB, MB><<<grid, 64 * parts, parts * NB * MB * 1024, s>>>(p, m);
    });
}

}  // namespace evamx

using namespace evamx;

extern "C" size_t evamx_w4_linear_workspace_bytes(int rows, int n_in)
{
    if (rows < 1 || rows > 65536 || n_in < 1 || n_in > EVAMX_W4_MAX_DIM) return 0;
    return w4_align((size_t)rows * 4) + w4_align((size_t)rows * w4_ceil(n_in, W4_TILE_K) * W4_TILE_K * 2);
}

extern "C" int evamx_w4_linear(const void* x, int x_dtype, int64_t x_stride, int rows, const evamx_w4_weight* w, const void* bias,
                               void* y, int64_t y_stride, void* workspace, size_t workspace_bytes, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!w4_weight_ok(w, "evamx_w4_linear")) return EVAMX_EINVAL;
    if (!x || !y || !workspace) { set_error("evamx_w4_linear: null pointer"); return EVAMX_EINVAL; }
    if (w->count != 1) { set_error("evamx_w4_linear: a stack of %d matrices", w->count); return EVAMX_EINVAL; }
    if (x_dtype != EVAMX_DTYPE_F16 && x_dtype != EVAMX_DTYPE_BF16) { set_error("evamx_w4_linear: x_dtype %d", x_dtype); return EVAMX_EINVAL; }
    if (rows < 1 || rows > 65536) { set_error("evamx_w4_linear: rows %d outside 1..65536", rows); return EVAMX_EINVAL; }
    if (x_stride < w->n_in || y_stride < w->n_out) { set_error("evamx_w4_linear: strides below the row lengths"); return EVAMX_EINVAL; }
    if ((uintptr_t)workspace & 15) { set_error("evamx_w4_linear: the workspace must be 16-byte aligned"); return EVAMX_EINVAL; }
    const size_t need = evamx_w4_linear_workspace_bytes(rows, w->n_in);
    if (workspace_bytes < need) { set_error("evamx_w4_linear: workspace %zu bytes < %zu", workspace_bytes, need); return EVAMX_ENOSPACE; }
    const hipStream_t s = (hipStream_t)stream;
    const W4Mat m = w4_mat(*w);
    const int parts = w4_parts(m.kt, m.nt);
    W4LinearParams p;
    p.x = x; p.x_stride = (size_t)x_stride; p.rows = rows; p.bf16 = x_dtype == EVAMX_DTYPE_BF16;
    p.aligned = (((uintptr_t)x | (uintptr_t)(2 * x_stride)) & 15) == 0;
    p.y_aligned = (((uintptr_t)y | (uintptr_t)(2 * y_stride)) & 15) == 0;
    p.bias = bias; p.y = y; p.y_stride = (size_t)y_stride; p.xh = nullptr; p.row_scale = nullptr;
    if (w4_stage_fits(rows, m.kt, parts)) {
        w4_dispatch(*w, [&](auto sg, auto zero) {
            w4_linear_few_kernel<decltype(sg)::value, decltype(zero)::value><<<m.nt, 64 * parts, w4_stage_bytes(rows, m.kt), s>>>(p, m);
        });
        return launched("w4_linear");
    }
    if (w4_rows_ready(x, x_dtype, x_stride, m.n_in)) {
        p.xh = (const w4_half*)x;
    } else {
        float* rs = (float*)workspace;
        w4_half* xh = (w4_half*)((char*)workspace + w4_align((size_t)rows * 4));
        w4_launch_rows(x, x_dtype, (size_t)x_stride, rows, w->n_in, xh, rs, s);
        p.xh = xh;
        p.row_scale = rs;
    }
    const long row_tiles = w4_ceil(rows, W4G_ROWS), col_tiles = w4_ceil(m.n_out, W4G_COLS);
    if (rows <= 16) {
        // 16 columns a workgroup while that gives a CU at most one (7168 -> 4096 at 5 and 16 rows: 10.9 and 14.5 us against 11.9 and
        // 15.2 with 32), else 32 on the same rows (7168 -> 5120: 12.0 and 15.3 against 14.4 and 22.3 with 16; 7168 -> 8192, whose
        // k-tiles are cut into four parts instead of eight: 16.4 and 18.0 against 14.5 and 21.3; 7168 -> 18432: 21.3 and 31 against
        // 26 and 42)
        if (m.nt <= W4_CUS) w4_launch_linear<1, 1>(p, m, *w, parts, s);
        else w4_launch_linear<2, 1>(p, m, *w, parts, s);
    } else if (row_tiles * col_tiles * m.kt >= 104l * m.kt + 600) {
        // The 64 x 256 tiles take about 1.5 us a k-tile and 5 for all of a round, the kernel below 0.014 us a tile and k-tile
        // (7168 -> 2048 at 200 rows: 80 us against 22; at 1024: 83 against 89; 2048 -> 7168 at 400: 38 and 36)
        w4_dispatch(*w, [&](auto sg, auto zero) {
            w4_linear_gemm_kernel<decltype(sg)::value, decltype(zero)::value>
                <<<8 * w4_ceil((int)(row_tiles * col_tiles), 8), 256, 0, s>>>(p, m, (int)row_tiles, (int)col_tiles);
        });
    } else if ((long)w4_ceil(m.nt, 2) * w4_ceil(rows, 32) <= W4_CUS) {
        // 32 columns by 32 rows while that gives a CU at most one workgroup (7168 -> 2048 at 17 rows: 12.6 us against 18.4, at 128:
        // 18.6 against 21.1), else 64 (7168 -> 2112 at 128: 33.4 against 21.4; 7168 -> 2048 at 200: 33.6 against 21.2)
        w4_launch_linear<2, 2>(p, m, *w, m.kt >= 8 ? 8 : parts, s);
    } else {
        w4_launch_linear<4, 2>(p, m, *w, parts < 4 ? parts : 4, s);
    }
    return launched("w4_linear");
}
