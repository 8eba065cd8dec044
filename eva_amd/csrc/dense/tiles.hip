// y = act(x W^T + b) + residual in tiles, and x's gradient D W, whose matrix has k over its rows.
#include <stdlib.h>

#include "linear.hpp"

namespace evamx_dense {

// WP by WQ by KW waves of 64 columns by 16 QB rows each.
template <class T, bool GATED, bool PTR, bool LOOSE, int WP, int WQ, int QB, int KW, int STAGES>
__device__ __forceinline__ void tile_product(const LinearParams& p, const Tile& t, char* lds)
{
    constexpr int PB = 4;
    typedef Gemm<T, PTR, false, WP, WQ, PB, QB, KW, STAGES, LOOSE> G;
    constexpr int COLS = GATED ? G::TP / 2 : G::TP;
    const uint16_t* w = p.w + (size_t)t.expert * p.w_expert_stride;
    typename G::P a;
    typename G::Q b;
    if constexpr (PTR) {
        a.init(w + t.col * COLS, p.w_stride, p.n_in, p.n_out - t.col * COLS, [](int n) { return n; });
    } else {
        a.init(w, p.w_stride, p.n_out, p.n_in, [&](int n) {
            if constexpr (!GATED) return COLS * t.col + n;
            const int j = COLS * t.col + 32 * (n >> 6) + (n & 31);
            return (n & 32) ? p.inter + j : j;                           // a wave's first 32 values are of the gate
        });
    }
    b.init(p.x + (size_t)t.row * p.x_stride, p.x_stride, t.have, p.n_in, [](int n) { return n; });
    f32x4 acc[PB][QB] = {};
    const int kt = (p.n_in + TILE_K - 1) / TILE_K, k0 = (int)((long)kt * blockIdx.y / p.splits), k1 = (int)((long)kt * (blockIdx.y + 1) / p.splits);
    if (!G::run(acc, a, b, lds, k0, k1)) return;
    const int lane = threadIdx.x & 63, wp = G::wp(), wq = G::wq();
    constexpr int CHUNKS = GATED ? 4 : 8, PASS = 64 / CHUNKS;            // eights of a row (SwiGLU: of the gate's half), rows a pass
    const int n = (GATED ? COLS * t.col + 32 * wp : COLS * t.col + 64 * wp) + 8 * (lane % CHUNKS);
    rows_of<PB, QB>(acc, lds, wq * WP + wp, [&](const float* mine, int first, int count) {
        for (int r0 = lane / CHUNKS; r0 < count; r0 += PASS) {
            const int r = 16 * QB * wq + first + r0;
            if (r >= t.have) break;
            float v[8], u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = mine[r0 * OUT_ROW + 8 * (lane % CHUNKS) + i];
                u[i] = GATED ? mine[r0 * OUT_ROW + 32 + 8 * (lane % CHUNKS) + i] : 0.0f;
            }
            if (p.splits > 1) {
                float* part = p.part + ((size_t)blockIdx.y * p.g.rows + t.row + r) * p.n_out + n;
                const int have = (GATED ? p.inter : p.n_out) - n;
                store_floats(part, v, have);
                if (GATED) store_floats(part + p.inter, u, have);
            } else {
                finish<T, GATED, 8>(p, t.expert, t.row + r, n, v, u);
            }
        }
    });
}

// SIZE: columns by rows of a workgroup's tile, 2: 256 by 256, 1: 256 by 128, 0: 128 by 128.
template <int SIZE>
struct TileShape {
    static constexpr int WP = SIZE ? 4 : 2, WQ = SIZE == 2 ? 2 : 1, KW = SIZE == 2 ? 1 : 2, STAGES = SIZE == 1 ? 3 : 2;
    static constexpr int TQ = 128 * WQ, THREADS = 64 * WP * WQ * KW;
};

template <class T, bool GATED, bool PTR, bool LOOSE, int SIZE>
__global__ __launch_bounds__(TileShape<SIZE>::THREADS, 2) void tiles_kernel(LinearParams p, int cols)
{
    typedef TileShape<SIZE> S;
    constexpr int WIDE = Gemm<T, PTR, false, S::WP, S::WQ, 4, 8, S::KW, S::STAGES, LOOSE>::LDS;
    constexpr int HALF = SIZE == 2 ? Gemm<T, PTR, false, 4, 1, 4, 8, 2, 3, LOOSE>::LDS : 0;
    __shared__ __attribute__((aligned(1024))) char lds[WIDE > HALF ? WIDE : HALF];
    Tile t;
    const bool any = find_tile<S::THREADS>(p.g, S::TQ, cols, blockIdx.x, (int*)lds, t);
    // each workgroup clears a share of the rows behind the last, beside the others' products
    if (p.g.starts) zero_rows(p.y, p.y_stride, GATED ? p.inter : p.n_out, p.g.end(), p.g.rows, blockIdx.x, gridDim.x);
    if (!any) return;
    __syncthreads();
    if constexpr (SIZE == 2) {
        if (t.have <= 64) return tile_product<T, GATED, PTR, LOOSE, 4, 1, 4, 2, 3>(p, t, lds);
        if (t.have <= 128) return tile_product<T, GATED, PTR, LOOSE, 4, 1, 8, 2, 3>(p, t, lds);
    }
    if constexpr (SIZE == 1) {
        if (t.have <= 64) return tile_product<T, GATED, PTR, LOOSE, 4, 1, 4, 2, 3>(p, t, lds);
    }
    tile_product<T, GATED, PTR, LOOSE, S::WP, S::WQ, 8, S::KW, S::STAGES>(p, t, lds);
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
        add_floats(v, part, cols - n);
        if (GATED) add_floats(u, part + p.inter, cols - n);
    }
    finish<T, GATED, 8>(p, 0, row, n, v, u);
}

template <class T, bool GATED, bool PTR, bool LOOSE, int SIZE>
static void launch_size(const LinearParams& p, hipStream_t s)
{
    typedef TileShape<SIZE> S;
    const int cols = ceil_div(GATED ? p.inter : p.n_out, GATED ? 32 * S::WP : 64 * S::WP);
    const int64_t work = most_row_tiles(p.g.rows, p.g.experts, p.g.starts, S::TQ) * cols;
    tiles_kernel<T, GATED, PTR, LOOSE, SIZE><<<dim3((unsigned)(8 * ceil_div(work, 8)), p.splits), S::THREADS, 0, s>>>(p, cols);
}

template <class T, bool GATED, bool PTR, bool LOOSE>
static void launch_by_size(const LinearParams& p, hipStream_t s)
{
    if (p.splits > 1 || LOOSE) return launch_size<T, GATED, PTR, LOOSE, 0>(p, s);
    if constexpr (!LOOSE) {
        const int64_t tiles = most_row_tiles(p.g.rows, p.g.experts, p.g.starts, 256) * ceil_div(p.n_out, 256);
        static const char* force = getenv("TILE_SIZE");
        const int size = force ? atoi(force) : p.g.starts ? 2 : tiles >= 200 ? 2 : tiles >= 100 ? 1 : 0;
        if (size == 2) launch_size<T, GATED, PTR, LOOSE, 2>(p, s);
        else if (size == 1) launch_size<T, GATED, PTR, LOOSE, 1>(p, s);
        else launch_size<T, GATED, PTR, LOOSE, 0>(p, s);
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
