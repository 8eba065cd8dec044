// y = act(x W^T + b) + residual for few rows an expert: the weights, which are most of what is read, go from memory to the matrix
// cores' operands directly.
#include "linear.hpp"

namespace evamx_dense {

// A workgroup takes 16 columns (SwiGLU: of the gate and of the up product) of up to 64 rows; its waves split the sum and meet in LDS.
// Eight, or four where the weights stream: there the workgroups are many (64 experts of 7168 -> 4096, a row each: 537 us against 550; but
// one row of 7168 -> 2048, 128 workgroups: 12.6 against 11.7).
constexpr int FEW_ROWS = 64;
constexpr int few_waves(int lie) { return lie == LIE_STREAM ? 4 : 8; }
constexpr bool few_whole(int lie) { return lie == LIE_16 || lie == LIE_STREAM; }     // 16-byte addresses

// 16 bytes at k of a row of n values. TAIL: the row may begin or end there; values behind its end are zeros.
template <int LIE, bool TAIL>
__device__ __forceinline__ u16x8 few_load(const uint16_t* row, int k, int n)
{
    if (!TAIL || k + 8 <= n) return *(const typename std::conditional<!few_whole(LIE), u16x8_loose, u16x8>::type*)(row + k);
    u16x8 x = (u16x8)(uint16_t)0;
    if (!few_whole(LIE)) {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (k + i < n) x[i] = row[k + i];
    }
    return x;
}

// A wave's operands of C steps from row on (this lane's chunk of the first one) where rows start at any value's address: whole words and
// a shift. The word behind a chunk is the first of the next lane's, lane + 16 of the same step or lane - 48 of the next one, and
// loaded for the last step alone (load8_shifted in their place: 13 rows, 5001 -> 2303, 15 us against 10).
template <int C>
struct FewShifted {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef u32x4 words __attribute__((aligned(4)));
    u32x4 v[C];
    uint32_t behind;
    int shift;

    __device__ __forceinline__ void load(const uint16_t* row)
    {
        const uint32_t* at = (const uint32_t*)((uintptr_t)row & ~(uintptr_t)3);
        shift = (int)((uintptr_t)row & 2) * 8;
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] = *(const words*)(at + 16 * i);
        behind = at[16 * (C - 1) + 4];
    }
    __device__ __forceinline__ void take(u16x8 (&out)[C])
    {
        const int lane = threadIdx.x & 63;
        uint32_t next[C + 1];
#pragma unroll
        for (int i = 0; i < C; ++i) next[i] = __builtin_amdgcn_ds_bpermute(4 * (lane + 16 & 63), v[i][0]);
        next[C] = behind;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const uint32_t end = lane < 48 ? next[i] : next[i + 1];
            u32x4 o;
            o[0] = __builtin_amdgcn_alignbit(v[i][1], v[i][0], shift);
            o[1] = __builtin_amdgcn_alignbit(v[i][2], v[i][1], shift);
            o[2] = __builtin_amdgcn_alignbit(v[i][3], v[i][2], shift);
            o[3] = __builtin_amdgcn_alignbit(end, v[i][3], shift);
            out[i] = __builtin_bit_cast(u16x8, o);
        }
    }
};

// Two steps of 16 rows of weights in whole lines (in halves of lines, 16 rows an instruction, the same loads take 312 us instead of 263
// at 25 experts of 7168 -> 4096; marked as not used again, 392 instead of 247): each load takes 64 values of eight rows, and lanes 8
// apart exchange what belongs to the other's row. first, second: this lane's chunk of row c % 8 and of row 8 + c % 8, 8 (g + 4 (c / 8))
// values into the steps.
template <int LIE>
__device__ __forceinline__ void few_lines(const uint16_t* first, const uint16_t* second, u16x8& step0, u16x8& step1)
{
#ifdef __HIP_DEVICE_COMPILE__
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 x, y, p, q;
    if constexpr (LIE == LIE_STREAM) {
        x = __builtin_nontemporal_load((const u32x4*)first);
        y = __builtin_nontemporal_load((const u32x4*)second);
    } else {
        x = *(const u32x4*)first;
        y = *(const u32x4*)second;
    }
    const bool low = (threadIdx.x & 8) == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t got = __builtin_amdgcn_update_dpp(0, low ? y[i] : x[i], 0x128, 0xf, 0xf, true);    // row_ror:8
        p[i] = low ? x[i] : got;
        q[i] = low ? got : y[i];
    }
    step0 = __builtin_bit_cast(u16x8, p);
    step1 = __builtin_bit_cast(u16x8, q);
#endif
}

template <class T, bool GATED, int LIE, int MB, int CB>
__device__ __forceinline__ void few_product(const LinearParams& p, const Tile& t, f32x4* part)
{
    constexpr int NB = GATED ? 2 * CB : CB, AHEAD = (NB + MB) <= 2 ? 8 : NB + MB <= 5 ? 4 : 2, WAVES = few_waves(LIE);
    constexpr bool LINES = few_whole(LIE);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const uint16_t* w = p.w + (size_t)t.expert * p.w_expert_stride;
    const uint16_t* a[NB];                                               // the up product's blocks behind the gate's
    const uint16_t* lines[LINES ? NB : 1][2];
    const uint16_t* x[MB];
    const int cols = GATED ? p.inter : p.n_out;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        const int n = 16 * (CB * t.col + b) + c, nn = n < cols ? n : cols - 1;
        a[b] = w + (size_t)nn * p.w_stride;
        if (GATED) a[NB - CB + b] = w + (size_t)(p.inter + nn) * p.w_stride;
        if constexpr (LINES) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = 16 * (CB * t.col + b) + 8 * h + (c & 7), row = at < cols ? at : cols - 1;
                lines[b][h] = w + (size_t)row * p.w_stride + 8 * g + 32 * (c >> 3);
                if (GATED) lines[NB - CB + b][h] = w + (size_t)(p.inter + row) * p.w_stride + 8 * g + 32 * (c >> 3);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int r = 16 * m + c;
        x[m] = p.x + (size_t)(t.row + (r < t.have ? r : t.have - 1)) * p.x_stride;
    }
    f32x4 acc[NB][MB] = {};
    // a wave's steps, in pairs: a line of 128 bytes
    const int steps = (p.n_in + 31) / 32, s1 = wave == WAVES - 1 ? steps : steps / 2 * (wave + 1) / WAVES * 2;
    int s = steps / 2 * wave / WAVES * 2;
    auto some = [&](auto count, auto tail) {
        constexpr int C = decltype(count)::value;
        constexpr bool TAIL = decltype(tail)::value;
        u16x8 wv[NB][C], xv[MB][C];
        if constexpr (LIE == LIE_2 && !TAIL) {
            FewShifted<C> wr[NB], xr[MB];
#pragma unroll
            for (int b = 0; b < NB; ++b) wr[b].load(a[b] + 32 * s + 8 * g);
#pragma unroll
            for (int m = 0; m < MB; ++m) xr[m].load(x[m] + 32 * s + 8 * g);
#pragma unroll
            for (int b = 0; b < NB; ++b) wr[b].take(wv[b]);
#pragma unroll
            for (int m = 0; m < MB; ++m) xr[m].take(xv[m]);
        } else if constexpr (LINES && !TAIL && C % 2 == 0) {
#pragma unroll
            for (int i = 0; i < C; i += 2) {
                const int k = 32 * (s + i);
#pragma unroll
                for (int b = 0; b < NB; ++b) few_lines<LIE>(lines[b][0] + k, lines[b][1] + k, wv[b][i], wv[b][i + 1]);
            }
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int m = 0; m < MB; ++m) xv[m][i] = few_load<LIE, TAIL>(x[m], 32 * (s + i) + 8 * g, p.n_in);
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int k = 32 * (s + i) + 8 * g;
#pragma unroll
                for (int b = 0; b < NB; ++b) wv[b][i] = few_load<LIE, TAIL>(a[b], k, p.n_in);
#pragma unroll
                for (int m = 0; m < MB; ++m) xv[m][i] = few_load<LIE, TAIL>(x[m], k, p.n_in);
            }
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < MB; ++m) acc[b][m] = T::mfma(wv[b][i], xv[m][i], acc[b][m]);
        s += C;
    };
    // steps that end within the rows; loads of shifted words also begin there, and reach two values further
    const int inside = (LIE == LIE_2 ? p.n_in - 2 : p.n_in) / 32, whole = inside < s1 ? inside : s1;
    if (LIE == LIE_2 && s == 0 && s < s1) some(std::integral_constant<int, 1>(), std::true_type());
    while (s + AHEAD <= whole) some(std::integral_constant<int, AHEAD>(), std::false_type());
    if (s + AHEAD / 2 <= whole) some(std::integral_constant<int, AHEAD / 2>(), std::false_type());
    while (s < whole) some(std::integral_constant<int, 1>(), std::false_type());
    while (s < s1) some(std::integral_constant<int, 1>(), std::true_type());
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m) part[((wave * NB + b) * MB + m) * 64 + lane] = acc[b][m];
    __syncthreads();
    for (int block = wave; block < CB * MB; block += WAVES) {
        const int m = block % MB, b = block / MB, r = 16 * m + c;
        if (r >= t.have) continue;
        Finish<T, GATED> end;
        end.init(p, t.expert, 16 * (CB * t.col + b) + 4 * g);
        const u16x4 res = end.residual(p, t.row + r);
        float v[4] = {}, u[4] = {};
        for (int q = 0; q < WAVES; ++q) {
            const f32x4 s = part[((q * NB + b) * MB + m) * 64 + lane], s2 = part[((q * NB + NB - CB + b) * MB + m) * 64 + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] += s[i];
                if (GATED) u[i] += s2[i];
            }
        }
        end.store(p, t.row + r, v, u, res);
    }
}

template <class T, bool GATED, int LIE, int CB>
__global__ __launch_bounds__(64 * few_waves(LIE)) void few_kernel(LinearParams p, int cols)
{
    extern __shared__ f32x4 part[];
    constexpr int WAVES = few_waves(LIE);
    __shared__ int scratch[2 + WAVES];
    Tile t = {0, 0, p.g.rows, (int)blockIdx.x};
    bool any = (int)blockIdx.x < cols;
    if (p.g.starts || p.g.rows > FEW_ROWS) {
        Tiles<64 * WAVES, FEW_ROWS> tiles;
        tiles.init(p.g, cols, scratch);
        any = tiles.find(blockIdx.x, t);
    }
    if (p.g.starts && p.g.upto == Groups::ALL) zero_rows(p.y, p.y_stride, GATED ? p.inter : p.n_out, p.g.end(), p.g.rows, blockIdx.x, gridDim.x);
    if (!any) return;
    if (t.have > 32) few_product<T, GATED, LIE, 4, CB>(p, t, part);
    else if (t.have > 16) few_product<T, GATED, LIE, 2, CB>(p, t, part);
    else few_product<T, GATED, LIE, 1, CB>(p, t, part);
}

template <class T, bool GATED, int LIE, int CB>
static void launch_few_as(const LinearParams& p, hipStream_t s)
{
    const int rows = p.g.rows < p.g.upto ? p.g.rows : p.g.upto;
    const int cols = ceil_div(GATED ? p.inter : p.n_out, 16 * CB), most = rows > 32 ? 4 : rows > 16 ? 2 : 1;
    const int64_t work = most_row_tiles(p.g, FEW_ROWS) * cols;
    few_kernel<T, GATED, LIE, CB><<<(unsigned)(8 * ceil_div(work, 8)), 64 * few_waves(LIE), (GATED ? 2 : 1) * CB * few_waves(LIE) * most * 1024, s>>>(p, cols);
}

int launch_few(const LinearParams& p, int dtype, int lie, hipStream_t s)
{
    // 32 columns a workgroup, which read the rows once for twice the weights, where that leaves a workgroup for most CUs (16 rows of
    // 2048 -> 7168: 9.6 us against 11.1, 64: 14.3 against 21; 7168 -> 2048: 21 and 40 against 16 and 35)
    const bool wide = !p.inter && p.g.rows > 8 && p.n_out >= 32 * CUS * 3 / 4;
    auto as = [&](auto type, auto gated, auto cb) {
        typedef decltype(type) T;
        constexpr bool G = decltype(gated)::value;
        constexpr int CB = decltype(cb)::value;
        if (lie == LIE_16) launch_few_as<T, G, LIE_16, CB>(p, s);
        else if (lie == LIE_STREAM) launch_few_as<T, G, LIE_STREAM, CB>(p, s);
        else if (lie == LIE_4) launch_few_as<T, G, LIE_4, CB>(p, s);
        else launch_few_as<T, G, LIE_2, CB>(p, s);
    };
    auto go = [&](auto type) {
        if (p.inter) as(type, std::true_type(), std::integral_constant<int, 1>());
        else if (wide) as(type, std::false_type(), std::integral_constant<int, 2>());
        else as(type, std::false_type(), std::integral_constant<int, 1>());
    };
    if (dtype == EVAMX_DTYPE_BF16) go(Bf16());
    else go(F16());
    return launched("linear");
}

}  // namespace evamx_dense
