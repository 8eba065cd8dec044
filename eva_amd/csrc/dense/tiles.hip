// y = act(x W^T + b) + residual in tiles, and x's gradient D W, whose matrix has k over its rows.
#include "linear.hpp"

namespace evamx_dense {

template <class T, bool GATED, bool PTR, bool LOOSE, int WP, int WQ, int QB>
__device__ __forceinline__ void tile_product(const LinearParams& p, const Tile& t, char* lds)
{
    constexpr int PB = 4;
    typedef Gemm<T, PTR, false, WP, WQ, PB, QB, LOOSE> G;
    constexpr int COLS = GATED ? G::TP / 2 : G::TP;
    const uint16_t* w = p.w + (size_t)t.expert * p.w_expert_stride;
    typename G::P a;
    typename G::Q b;
    if constexpr (PTR) {
        a.init(w + t.col * COLS, p.w_stride, p.n_in, p.n_out - t.col * COLS, [](int n) { return n; });
    } else {
        a.init(w, p.w_stride, p.n_out, p.n_in, [&](int n) {
            const int in32 = 8 * ((n & 15) >> 2) + 4 * ((n >> 4) & 1) + (n & 3);
            if constexpr (GATED) {
                const int j = COLS * t.col + 32 * (n >> 6) + in32;
                return (n & 32) ? p.inter + j : j;
            } else {
                return COLS * t.col + (n & ~31) + in32;
            }
        });
    }
    b.init(p.x + (size_t)t.row * p.x_stride, p.x_stride, t.have, p.n_in, [](int n) { return n; });
    f32x4 acc[PB][QB] = {};
    const int kt = (p.n_in + TILE_K - 1) / TILE_K, k0 = (int)((long)kt * blockIdx.y / p.splits), k1 = (int)((long)kt * (blockIdx.y + 1) / p.splits);
    G::run(acc, a, b, lds, k0, k1);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int wp = wave % WP, wq = wave / WP;
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        const int r = 16 * (QB * wq + j) + c;
        if (r >= t.have) continue;
        const int row = t.row + r;
        float v[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[h][i] = acc[2 * h + i / 4][j][i % 4];
        if (p.splits > 1) {
            float* part = p.part + ((size_t)blockIdx.y * p.g.rows + row) * p.n_out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = GATED ? COLS * t.col + 32 * wp + 8 * g : COLS * t.col + 64 * wp + 32 * h + 8 * g;
                const int end = GATED ? p.inter : p.n_out;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (n + i < end) part[(GATED && h ? p.inter : 0) + n + i] = v[h][i];
            }
        } else if constexpr (GATED) {
            finish<T, true, 8>(p, t.expert, row, COLS * t.col + 32 * wp + 8 * g, v[0], v[1]);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) finish<T, false, 8>(p, t.expert, row, COLS * t.col + 64 * wp + 32 * h + 8 * g, v[h], v[h]);
        }
    }
}

template <class T, bool GATED, bool PTR, bool LOOSE, int WP, int WQ, int QB>
__global__ __launch_bounds__(64 * WP * WQ, 2) void tiles_kernel(LinearParams p, int cols, int work)
{
    constexpr int THREADS = 64 * WP * WQ, TQ = 16 * QB * WQ;
    __shared__ __attribute__((aligned(1024))) char lds[Gemm<T, PTR, false, WP, WQ, 4, QB, LOOSE>::LDS];
    if ((int)blockIdx.x >= work) {
        if (p.g.starts) zero_rows(p.y, p.y_stride, GATED ? p.inter : p.n_out, p.g.end(), p.g.rows, blockIdx.x - work, gridDim.x - work);
        return;
    }
    Tile t;
    int row_tiles;
    if (!find_tile<THREADS>(p.g, TQ, cols, blockIdx.x, (int*)lds, t, row_tiles)) return;
    __syncthreads();
    if constexpr (QB == 8) {
        if (t.have <= TQ / 4) return tile_product<T, GATED, PTR, LOOSE, WP, WQ, 2>(p, t, lds);
        if (t.have <= TQ / 2) return tile_product<T, GATED, PTR, LOOSE, WP, WQ, 4>(p, t, lds);
    }
    tile_product<T, GATED, PTR, LOOSE, WP, WQ, QB>(p, t, lds);
}

// Sums of the splits, and what follows a sum.
template <class T, bool GATED>
__global__ __launch_bounds__(256) void join_kernel(LinearParams p)
{
    const int cols = GATED ? p.inter : p.n_out, per = (cols + 7) / 8;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(at / per), n = (int)(at % per) * 8;
    if (row >= p.g.rows) return;
    float v[8] = {}, u[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        const float* part = p.part + ((size_t)s * p.g.rows + row) * p.n_out + n;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < cols) {
                v[i] += part[i];
                if (GATED) u[i] += part[p.inter + i];
            }
    }
    finish<T, GATED, 8>(p, 0, row, n, v, u);
}

constexpr int TAIL_GROUPS = 256;

template <class T, bool GATED, bool PTR, bool LOOSE, int WP, int WQ, int QB>
static void launch_config(const LinearParams& p, hipStream_t s)
{
    constexpr int TQ = 16 * QB * WQ, COLS = GATED ? 32 * WP : 64 * WP;
    const int cols = ceil_div(GATED ? p.inter : p.n_out, COLS);
    const int64_t work = 8 * (int64_t)ceil_div(most_row_tiles(p.g.rows, p.g.experts, p.g.starts, TQ) * cols, 8);
    tiles_kernel<T, GATED, PTR, LOOSE, WP, WQ, QB>
        <<<dim3((unsigned)(work + (p.g.starts ? TAIL_GROUPS : 0)), p.splits), 64 * WP * WQ, 0, s>>>(p, cols, (int)work);
}

template <class T, bool GATED, bool PTR, bool LOOSE>
static void launch_by_size(const LinearParams& p, hipStream_t s)
{
    if (p.splits > 1) {
        launch_config<T, GATED, PTR, LOOSE, 2, 2, 4>(p, s);
    } else if constexpr (LOOSE) {
        launch_config<T, GATED, PTR, LOOSE, 2, 2, 4>(p, s);
    } else {
        const int64_t tiles = most_row_tiles(p.g.rows, p.g.experts, p.g.starts, 256) * ceil_div(p.n_out, 256);
        if (tiles >= CUS / 2) launch_config<T, GATED, PTR, LOOSE, 4, 2, 8>(p, s);
        else launch_config<T, GATED, PTR, LOOSE, 2, 2, 4>(p, s);
    }
}

template <class T>
static void launch_typed(const LinearParams& p, bool transposed, bool loose, hipStream_t s)
{
    if (transposed) {
        if (loose) launch_by_size<T, false, true, true>(p, s);
        else launch_by_size<T, false, true, false>(p, s);
    } else if (p.inter) {
        if (loose) launch_by_size<T, true, false, true>(p, s);
        else launch_by_size<T, true, false, false>(p, s);
    } else {
        if (loose) launch_by_size<T, false, false, true>(p, s);
        else launch_by_size<T, false, false, false>(p, s);
    }
}

int launch_tiles(const LinearParams& p, int dtype, bool transposed, bool loose, hipStream_t s)
{
    if (dtype == EVAMX_DTYPE_BF16) launch_typed<Bf16>(p, transposed, loose, s);
    else launch_typed<F16>(p, transposed, loose, s);
    if (p.splits > 1) return launch_join(p, dtype, s);
    return launched("linear");
}

int launch_join(const LinearParams& p, int dtype, hipStream_t s)
{
    const unsigned grid = (unsigned)ceil_div((int64_t)p.g.rows * ceil_div(p.inter ? p.inter : p.n_out, 8), 256);
    if (dtype == EVAMX_DTYPE_BF16) {
        if (p.inter) join_kernel<Bf16, true><<<grid, 256, 0, s>>>(p);
        else join_kernel<Bf16, false><<<grid, 256, 0, s>>>(p);
    } else {
        if (p.inter) join_kernel<F16, true><<<grid, 256, 0, s>>>(p);
        else join_kernel<F16, false><<<grid, 256, 0, s>>>(p);
    }
    return launched("linear");
}

}  // namespace evamx_dense
