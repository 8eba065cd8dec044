// y = act(x W^T + b) + residual for few rows an expert: the weights, which are most of what is read, go from memory to the matrix
// cores' operands directly.
#include "linear.hpp"

namespace evamx_dense {

// A workgroup takes 16 columns (SwiGLU: of the gate and of the up product) of up to 64 rows; its waves split the sum and meet in LDS.
constexpr int FEW_WAVES = 8, FEW_THREADS = 64 * FEW_WAVES, FEW_ROWS = 64;

// 16 bytes at k of a row of n values; values behind the row's end are zeros.
template <bool LOOSE>
__device__ __forceinline__ u16x8 few_load(const uint16_t* row, int k, int n)
{
    if (!LOOSE || k + 8 <= n) {
        if (!LOOSE && k >= n) return (u16x8)(uint16_t)0;
        return *(const typename std::conditional<LOOSE, u16x8_loose, u16x8>::type*)(row + k);
    }
    u16x8 x = (u16x8)(uint16_t)0;
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (k + i < n) x[i] = row[k + i];
    return x;
}

template <class T, bool GATED, bool LOOSE, int MB>
__device__ __forceinline__ void few_product(const LinearParams& p, const Tile& t, f32x4* part)
{
    constexpr int NB = GATED ? 2 : 1, AHEAD = MB == 1 ? 8 : MB == 2 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const uint16_t* w = p.w + (size_t)t.expert * p.w_expert_stride;
    const uint16_t* a[NB];
    const uint16_t* x[MB];
    const int n = 16 * t.col + c, cols = GATED ? p.inter : p.n_out, nn = n < cols ? n : cols - 1;
    a[0] = w + (size_t)nn * p.w_stride;
    if (GATED) a[NB - 1] = w + (size_t)(p.inter + nn) * p.w_stride;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int r = 16 * m + c;
        x[m] = p.x + (size_t)(t.row + (r < t.have ? r : t.have - 1)) * p.x_stride;
    }
    f32x4 acc[NB][MB] = {};
    const int steps = (p.n_in + 31) / 32, s1 = (int)((long)steps * (wave + 1) / FEW_WAVES);
    int s = (int)((long)steps * wave / FEW_WAVES);
    auto some = [&](auto count) {
        constexpr int C = decltype(count)::value;
        u16x8 wv[C][NB], xv[C][MB];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int k = 32 * (s + i) + 8 * g;
#pragma unroll
            for (int b = 0; b < NB; ++b) wv[i][b] = few_load<LOOSE>(a[b], k, p.n_in);
#pragma unroll
            for (int m = 0; m < MB; ++m) xv[i][m] = few_load<LOOSE>(x[m], k, p.n_in);
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < MB; ++m) acc[b][m] = T::mfma(wv[i][b], xv[i][m], acc[b][m]);
        s += C;
    };
    while (s + AHEAD <= s1) some(std::integral_constant<int, AHEAD>());
    while (s < s1) some(std::integral_constant<int, 1>());
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m) part[((wave * NB + b) * MB + m) * 64 + lane] = acc[b][m];
    __syncthreads();
    for (int m = wave; m < MB; m += FEW_WAVES) {
        const int r = 16 * m + c;
        if (r >= t.have) continue;
        float v[NB][4] = {};
        for (int q = 0; q < FEW_WAVES; ++q)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[b][i] += part[((q * NB + b) * MB + m) * 64 + lane][i];
        finish<T, GATED, 4>(p, t.expert, t.row + r, 16 * t.col + 4 * g, v[0], v[NB - 1]);
    }
}

template <class T, bool GATED, bool LOOSE>
__global__ __launch_bounds__(FEW_THREADS) void few_kernel(LinearParams p, int cols)
{
    extern __shared__ f32x4 part[];
    Tile t;
    const bool any = find_tile<FEW_THREADS>(p.g, FEW_ROWS, cols, blockIdx.x, (int*)part, t);
    if (p.g.starts) zero_rows(p.y, p.y_stride, GATED ? p.inter : p.n_out, p.g.end(), p.g.rows, blockIdx.x, gridDim.x);
    if (!any) return;
    __syncthreads();
    if (t.have > 32) few_product<T, GATED, LOOSE, 4>(p, t, part);
    else if (t.have > 16) few_product<T, GATED, LOOSE, 2>(p, t, part);
    else few_product<T, GATED, LOOSE, 1>(p, t, part);
}

template <class T, bool GATED, bool LOOSE>
static void launch_few_as(const LinearParams& p, hipStream_t s)
{
    const int cols = ceil_div(GATED ? p.inter : p.n_out, 16), most = p.g.rows > 32 ? 4 : p.g.rows > 16 ? 2 : 1;
    const int64_t work = most_row_tiles(p.g.rows, p.g.experts, p.g.starts, FEW_ROWS) * cols;
    few_kernel<T, GATED, LOOSE><<<(unsigned)(8 * ceil_div(work, 8)), FEW_THREADS, (GATED ? 2 : 1) * FEW_WAVES * most * 1024, s>>>(p, cols);
}

int launch_few(const LinearParams& p, int dtype, bool loose, hipStream_t s)
{
    auto go = [&](auto type) {
        typedef decltype(type) T;
        if (p.inter) {
            if (loose) launch_few_as<T, true, true>(p, s);
            else launch_few_as<T, true, false>(p, s);
        } else {
            if (loose) launch_few_as<T, false, true>(p, s);
            else launch_few_as<T, false, false>(p, s);
        }
    };
    if (dtype == EVAMX_DTYPE_BF16) go(Bf16());
    else go(F16());
    return launched("linear");
}

}  // namespace evamx_dense
