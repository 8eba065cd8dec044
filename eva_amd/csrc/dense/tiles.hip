// y = act(x W^T + b) + residual in tiles, and x's gradient D W, whose matrix has k over its rows. With few rows an expert the weights
// are what is read: 32 experts of 128 rows, 7168 -> 4096, 1.9 GB: 432 us, 4.4 TB/s.
#include "linear.hpp"

namespace evamx_dense {

// WP by WQ by KW waves of 64 columns by 16 QB rows each.
template <class T, bool GATED, bool PTR, int WP, int WQ, int QB, int KW, int STAGES>
struct TileProduct {
    static constexpr int PB = 4;
    typedef Gemm<T, PTR, false, WP, WQ, PB, QB, KW, STAGES> G;
    static constexpr int COLS = GATED ? G::TP / 2 : G::TP;

    // Results that are the sums and a bias alone, or SwiGLU's of them, in whole columns: from the registers.
    static __device__ __forceinline__ bool plain(const LinearParams& p, const Tile& t)
    {
        return p.splits == 1 && !p.residual && !p.pre && (GATED || p.act == EVAMX_ACT_NONE) && COLS * (t.col + 1) <= (GATED ? p.inter : p.n_out);
    }
    template <bool STREAM>
    static __device__ __forceinline__ void store_plain(const LinearParams& p, const Tile& t, const f32x4 (&acc)[PB][QB])
    {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        const bool all = t.have == G::TQ;
        f32x4 bias[PB] = {};
        if (p.bias) {
            const uint16_t* b = p.bias + (size_t)t.expert * p.n_out + COLS * t.col + (GATED ? 32 : 64) * G::wp() + 4 * g;
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const u16x4 x = *(const u16x4_loose*)(b + (GATED && i >= 2 ? p.inter - 32 : 0) + 16 * i);
                bias[i] = f32x4{T::get(x[0]), T::get(x[1]), T::get(x[2]), T::get(x[3])};
            }
        }
        if constexpr (GATED) {
            const int r0 = 16 * QB * G::wq() + c;
            uint16_t* at = p.y + (size_t)(t.row + r0) * p.y_stride + COLS * t.col + 32 * G::wp() + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                f32x4 y[2];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[b][i] = swiglu(acc[b][j][i] + bias[b][i], acc[2 + b][j][i] + bias[2 + b][i], p.limit);
                const u16x8 v = paired<T>(y[0], y[1]);
                if (all || r0 + 16 * j < t.have) store16<STREAM>(at + (size_t)(16 * j) * p.y_stride, v);
            }
        } else {
            const int r0 = 16 * QB * G::wq() + (c & 7);
            uint16_t* at = p.y + (size_t)(t.row + r0) * p.y_stride + COLS * t.col + 64 * G::wp() + 32 * (c >> 3) + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                const f32x4 sums[4] = {acc[0][j] + bias[0], acc[1][j] + bias[1], acc[2][j] + bias[2], acc[3][j] + bias[3]};
                u16x8 v[2];
                lined<T>(sums, v);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (all || r0 + 16 * j + 8 * i < t.have) store16<STREAM>(at + (size_t)(16 * j + 8 * i) * p.y_stride, v[i]);
            }
        }
    }
    // All others, by way of LDS, eight (four) rows of a lane at a time: their residuals are asked for with those before (one row at a time:
    // 300 rows of 2048 -> 7168 with bias, GELU and residual 59 us).
    static __device__ __forceinline__ void store(const LinearParams& p, const Tile& t, const f32x4 (&acc)[PB][QB], char* lds)
    {
        constexpr int FOURS = GATED ? 8 : 16, PASS = 64 / FOURS, BATCH = GATED ? 4 : 8;    // fours of a row (SwiGLU: of the gate's half), rows a pass
        const int lane = threadIdx.x & 63, wp = G::wp(), in = 4 * (lane % FOURS), cols = GATED ? p.inter : p.n_out;
        const int n = (GATED ? COLS * t.col + 32 * wp : COLS * t.col + 64 * wp) + in, r0 = 16 * QB * G::wq() + lane / FOURS;
        Finish<T, GATED> end;
        u16x4 next[BATCH] = {};
        auto ask = [&](int r) {
            if (p.residual && r - r0 < 16 * QB) {
#pragma unroll
                for (int i = 0; i < BATCH; ++i)
                    if (r + PASS * i < t.have) next[i] = end.residual(p, t.row + r + PASS * i);
            }
        };
        if (p.splits == 1) {
            end.init(p, t.expert, n);
            ask(r0);
        }
        rows_of<PB, QB>(acc, lds, G::wq() * WP + wp, [&](const float* mine, int first, int count) {
#pragma unroll 1
            for (int b = 0; b < count; b += PASS * BATCH) {
                f32x4 x[BATCH], y[BATCH];
                u16x4 res[BATCH];
                const int r = r0 + first + b;
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const float* at = mine + (b + lane / FOURS + PASS * i) * OUT_ROW + in;
                    x[i] = *(const f32x4*)at;
                    y[i] = *(const f32x4*)(at + (GATED ? 32 : 0));
                    res[i] = next[i];
                }
                if (p.splits == 1) ask(r + PASS * BATCH);
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int row = t.row + r + PASS * i;
                    if (r + PASS * i >= t.have) break;
                    float v[4] = {x[i][0], x[i][1], x[i][2], x[i][3]}, u[4] = {y[i][0], y[i][1], y[i][2], y[i][3]};
                    if (p.splits > 1) {
                        float* part = p.part + ((size_t)blockIdx.y * p.g.rows + row) * p.n_out + n;
                        store_floats(part, v, cols - n);
                        if (GATED) store_floats(part + p.inter, u, cols - n);
                    } else {
                        end.store(p, row, v, u, res[i]);
                    }
                }
            }
        });
    }

    static __device__ __forceinline__ void take(const LinearParams& p, const Tile& t, char* lds)
    {
        const uint16_t* w = p.w + (size_t)t.expert * p.w_expert_stride;
        typename G::P a;
        typename G::Q b;
        if constexpr (PTR) {
            a.init(w + t.col * COLS, p.w_stride, p.n_in, p.w_cols - t.col * COLS, [](int n) { return n; });
        } else if constexpr (GATED) {
            a.init(w, p.w_stride, p.n_out, p.w_cols, [&](int n) {           // a wave's first 32 values are of the gate
                const int j = COLS * t.col + 32 * (n >> 6) + (n & 31);
                return (n & 32) ? p.inter + j : j;
            });
        } else {
            const int n0 = COLS * t.col;
            a.init(w + (size_t)n0 * p.w_stride, p.w_stride, p.n_out - n0 < COLS ? p.n_out - n0 : COLS, p.w_cols, [](int n) { return n; });
        }
        b.init(p.x + (size_t)t.row * p.x_stride, p.x_stride, t.have, p.x_cols, [](int n) { return n; });
        const int kt = (p.n_in + TILE_K - 1) / TILE_K;
        const int k0 = p.splits > 1 ? (int)((long)kt * blockIdx.y / p.splits) : 0, k1 = p.splits > 1 ? (int)((long)kt * (blockIdx.y + 1) / p.splits) : kt;
        f32x4 acc[PB][QB] = {};
        G::begin(a, b, lds, k0, k1);
        if (!G::run(acc, a, b, lds, k0, k1)) return;
        if (!plain(p, t)) store(p, t, acc, lds);
        else if (p.stream) store_plain<true>(p, t, acc);
        else store_plain<false>(p, t, acc);
    }
};

// A workgroup's tile: 256 columns by 256 rows, or 128 by 128, whose waves take half a k-tile each: four, or, where no two workgroups
// share a CU, eight (2000 rows, x's gradient of 2048 -> 5120: 54.6 us against 57.9; 128 rows of 4096 -> 4096: 19.6 against 21.3).
template <int SIZE>
struct TileShape {
    static constexpr bool BIG = SIZE == TILES_256;
    static constexpr int WP = BIG ? 4 : 2, WQ = SIZE == TILES_128 ? 1 : 2, KW = BIG ? 1 : 2, QB = SIZE == TILES_128_ALONE ? 4 : 8;
    static constexpr int TQ = 16 * QB * WQ, THREADS = 64 * WP * WQ * KW;
};

template <class T, bool GATED, bool PTR, int SIZE>
__global__ __launch_bounds__(TileShape<SIZE>::THREADS, 2) void tiles_kernel(LinearParams p, int cols)
{
    typedef TileShape<SIZE> S;
    typedef TileProduct<T, GATED, PTR, S::WP, S::WQ, S::QB, S::KW, 2> Whole;
    // an expert's last rows: waves of half a k-tile, three k-tiles in LDS (32 experts of 128 rows, 7168 -> 4096: 438 us against 530
    // with the waves of the whole tile)
    typedef TileProduct<T, GATED, PTR, 4, 1, 8, 2, 3> Half;
    typedef TileProduct<T, GATED, PTR, 4, 1, 4, 2, 3> Quarter;
    __shared__ __attribute__((aligned(1024))) char lds[S::BIG && Half::G::LDS > Whole::G::LDS ? Half::G::LDS : Whole::G::LDS];
    Tile t;
    bool any;
    {
        Tiles<S::THREADS, S::TQ> tiles;
        tiles.init(p.g, cols, (int*)lds);
        any = tiles.find(blockIdx.x, t);
    }
    // each workgroup clears a share of the rows behind the last, beside the others' products
    if (p.g.starts) zero_rows(p.y, p.y_stride, GATED ? p.inter : p.n_out, p.g.end(), p.g.rows, blockIdx.x, gridDim.x);
    if (!any) return;
    __syncthreads();
    if constexpr (S::BIG) {
        if (t.have <= 64) return Quarter::take(p, t, lds);
        if (t.have <= 128) return Half::take(p, t, lds);
    }
    Whole::take(p, t, lds);
}

// Sums of the splits, and what follows a sum (16 rows of 4096 values in 16 parts: 3.8 us).
template <class T, bool GATED>
__global__ __launch_bounds__(256) void join_kernel(LinearParams p)
{
    const int cols = GATED ? p.inter : p.n_out, per = (cols + 3) / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(at / per), n = (int)(at % per) * 4;
    if (row >= p.g.rows) return;
    Finish<T, GATED> end;
    float v[4] = {}, u[4] = {};
    end.init(p, 0, n);
    const u16x4 res = end.residual(p, row);
    const float* part = p.part + (size_t)row * p.n_out + n;
    const size_t next = (size_t)p.g.rows * p.n_out;
    if (n + 4 <= cols) {
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) {
            add_floats(v, part + s * next, 4);
            if (GATED) add_floats(u, part + s * next + p.inter, 4);
        }
    } else {
        for (int s = 0; s < p.splits; ++s) {
            add_floats(v, part + s * next, cols - n);
            if (GATED) add_floats(u, part + s * next + p.inter, cols - n);
        }
    }
    end.store(p, row, v, u, res);
}

template <class T, bool GATED, bool PTR, int SIZE>
static void launch_size(const LinearParams& p, hipStream_t s)
{
    typedef TileShape<SIZE> S;
    const int cols = ceil_div(GATED ? p.inter : p.n_out, GATED ? 32 * S::WP : 64 * S::WP);
    // one at least, where few.hip takes all experts there can be, for the rows behind the last
    const int64_t most = most_row_tiles(p.g, S::TQ) * cols, work = 8 * (int64_t)ceil_div(most < 1 ? 1 : most, 8);
    tiles_kernel<T, GATED, PTR, SIZE><<<dim3((unsigned)work, p.splits), S::THREADS, 0, s>>>(p, cols);
}

template <class T, bool GATED, bool PTR>
static void launch_by_size(const LinearParams& p, hipStream_t s)
{
    const int64_t work = most_row_tiles(p.g, 128) * ceil_div(GATED ? p.inter : p.n_out, GATED ? 64 : 128) * p.splits;
    if (p.size == TILES_256) launch_size<T, GATED, PTR, TILES_256>(p, s);
    else if (work <= CUS) launch_size<T, GATED, PTR, TILES_128_ALONE>(p, s);
    else launch_size<T, GATED, PTR, TILES_128>(p, s);
}

template <class T>
static void launch_typed(const LinearParams& p, bool transposed, hipStream_t s)
{
    if (transposed) launch_by_size<T, false, true>(p, s);
    else if (p.inter) launch_by_size<T, true, false>(p, s);
    else launch_by_size<T, false, false>(p, s);
}

int launch_tiles(const LinearParams& p, int dtype, bool transposed, hipStream_t s)
{
    if (dtype == EVAMX_DTYPE_BF16) launch_typed<Bf16>(p, transposed, s);
    else launch_typed<F16>(p, transposed, s);
    if (p.splits > 1) return launch_join(p, dtype, s);
    return launched("linear");
}

int launch_join(const LinearParams& p, int dtype, hipStream_t s)
{
    const unsigned grid = (unsigned)ceil_div((int64_t)p.g.rows * ceil_div(p.inter ? p.inter : p.n_out, 4), 256);
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
