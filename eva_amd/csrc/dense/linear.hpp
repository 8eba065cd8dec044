// Forward products and the rows' gradients: parameters, and what happens to a row's results.
#pragma once
#include "gemm.hpp"

namespace evamx_dense {

struct LinearParams {
    const uint16_t* x;
    const uint16_t* w;
    const uint16_t* bias;
    const uint16_t* residual;
    uint16_t* y;
    float* pre;
    size_t x_stride, w_stride, w_expert_stride, residual_stride, y_stride;
    Groups g;
    int n_in, n_out;             // of the product: k is 0 .. n_in - 1
    int x_cols, w_cols;          // values in a row of x and w in tiles: multiples of 8, zeros behind the last
    int inter;                   // SwiGLU: n_out / 2, else 0
    int act;
    float limit;
    float* part;                 // [splits][rows][n_out] partial sums, or NULL
    int size, splits;            // of the tiles (plan_of)
    bool stream;                 // y is more than the last-level cache holds (48000 rows of 7168, 690 MB: 710 us against 718)
};

// Tiles of 256 by 256, one workgroup a CU, or of 128 by 128, two a CU or (chosen at the launch) one, and the parts a sum is cut into.
enum { TILES_128 = 0, TILES_256 = 1, TILES_128_ALONE = 2 };
struct Plan {
    int size, splits;
};
// For a result of rows by cols that sums k values: the plan of the least time as measured for both kinds of tiles. A k-tile of 64 takes
// a 256 by 256 tile 1.15 us, 1.5 with all CUs at work, and a 128 by 128 one 0.58, with two on every CU 0.85; a tile's begin and end 5
// and 4 us; no less than what is read at 4.9 TB/s (by 144 workgroups 2.6, 288 3.8); a cut sum 7 us more for the join, and its way
// through memory at 2.9 TB/s. (us: 1024 rows of 4096 -> 4096 in 128 by 128 tiles 43, cut in two 45, in four 58, in 256 by 256 tiles 79,
// 56 and 49; 128 rows 39, 29, 22 and 51, 36, 26.)
Plan plan_of(int64_t rows, int64_t cols, int64_t k);

// Eight values at p of a row, or as many as there are.
__device__ __forceinline__ void load8(float (&v)[8], const uint16_t* p, int have, bool bf16)
{
    u16x8 x = (u16x8)(uint16_t)0;
    if (have >= 8) {
        x = *(const u16x8_loose*)p;
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < have) x[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16 ? Bf16::get(x[i]) : F16::get(x[i]);
}

// What follows a sum, for four consecutive columns from n on, of any rows of an expert. v as summed, for SwiGLU the gate's, u the up
// product's. What it reads is asked for ahead of the stores, since requests end in their order: read in between, 2000 rows of 2048
// -> 5120 with bias, activation and its input kept take 69 us instead of 62.
template <class T, bool GATED>
struct Finish {
    int n, have;
    float bias[4], bias_up[4];

    __device__ __forceinline__ u16x4 get(const uint16_t* from) const
    {
        if (have >= 4) return *(const u16x4_loose*)from;
        u16x4 x = {};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < have) x[i] = from[i];
        return x;
    }
    __device__ __forceinline__ void init(const LinearParams& p, int expert, int column)
    {
        n = column;
        have = (GATED ? p.inter : p.n_out) - n;
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = bias_up[i] = 0.0f;
        if (p.bias && have > 0) {
            const uint16_t* b = p.bias + (size_t)expert * p.n_out + n;
            const u16x4 x = get(b), y = get(b + (GATED ? p.inter : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bias[i] = T::get(x[i]);
                bias_up[i] = T::get(y[i]);
            }
        }
    }
    __device__ __forceinline__ u16x4 residual(const LinearParams& p, int row) const
    {
        return p.residual && have > 0 ? get(p.residual + (size_t)row * p.residual_stride + n) : u16x4{};
    }
    __device__ __forceinline__ void store(const LinearParams& p, int row, float (&v)[4], float (&u)[4], u16x4 res) const
    {
        if (have <= 0) return;
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] += bias[i];
                if (GATED) u[i] += bias_up[i];
            }
        }
        if (p.pre) {
            float* at = p.pre + (size_t)row * p.n_out + n;
            store_floats(at, v, have);
            if (GATED) store_floats(at + p.inter, u, have);
        }
        if (GATED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = swiglu(v[i], u[i], p.limit);
        } else {
            activate(v, p.act);
        }
        u16x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = T::put(p.residual ? v[i] + T::get(res[i]) : v[i]);
        uint16_t* y = p.y + (size_t)row * p.y_stride + n;
        if (have >= 4) {
            *(u16x4_loose*)y = o;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < have) y[i] = o[i];
        }
    }
};

int launch_tiles(const LinearParams& p, int dtype, bool transposed, hipStream_t s);
// How x and w lie: 16-byte addresses and rows, whole words, or single values.
enum { LIE_16 = 0, LIE_4 = 1, LIE_2 = 2, LIE_STREAM = 3 };
int launch_few(const LinearParams& p, int dtype, int lie, hipStream_t s);
// Rows of n values (rows of each of `count` matrices) to rows of a multiple of 8, zeros behind the last.
int launch_pad(const uint16_t* from, size_t stride, size_t matrix_stride, int rows, int count, int n, uint16_t* to, hipStream_t s);
int launch_join(const LinearParams& p, int dtype, hipStream_t s);

}  // namespace evamx_dense
