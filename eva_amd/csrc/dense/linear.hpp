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

// Tiles of 256 by 256, one workgroup a CU, or of 128 by 128, two a CU, and the parts a sum is cut into.
enum { TILES_128 = 0, TILES_256 = 1 };
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

// Four consecutive results at column n of row `row`: v as summed, for SwiGLU the gate's, u the up product's.
template <class T, bool GATED>
__device__ __forceinline__ void finish(const LinearParams& p, int expert, int row, int n, float (&v)[4], float (&u)[4])
{
    const int cols = GATED ? p.inter : p.n_out, have = cols - n;
    if (have <= 0) return;
    auto get = [&](const uint16_t* from, float (&out)[4]) {
        if (have >= 4) {
            const u16x4 x = *(const u16x4_loose*)from;
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = T::get(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = i < have ? T::get(from[i]) : 0.0f;
        }
    };
    float t[4];
    if (p.bias) {
        const uint16_t* b = p.bias + (size_t)expert * p.n_out + n;
        get(b, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
        if (GATED) {
            get(b + p.inter, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] += t[i];
        }
    }
    if (p.pre) {
        float* at = p.pre + (size_t)row * p.n_out + n;
        store_floats(at, v, have);
        if (GATED) store_floats(at + p.inter, u, have);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = GATED ? swiglu(v[i], u[i], p.limit) : activate(v[i], p.act);
    if (p.residual) {
        get(p.residual + (size_t)row * p.residual_stride + n, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
    }
    uint16_t* y = p.y + (size_t)row * p.y_stride + n;
    if (have >= 4) {
        u16x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = T::put(v[i]);
        *(u16x4_loose*)y = o;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < have) y[i] = T::put(v[i]);
    }
}

int launch_tiles(const LinearParams& p, int dtype, bool transposed, hipStream_t s);
// How x and w lie: 16-byte addresses and rows, whole words, or single values.
enum { LIE_16 = 0, LIE_4 = 1, LIE_2 = 2, LIE_STREAM = 3 };
int launch_few(const LinearParams& p, int dtype, int lie, hipStream_t s);
// Rows of n values (rows of each of `count` matrices) to rows of a multiple of 8, zeros behind the last.
int launch_pad(const uint16_t* from, size_t stride, size_t matrix_stride, int rows, int count, int n, uint16_t* to, hipStream_t s);
int launch_join(const LinearParams& p, int dtype, hipStream_t s);

}  // namespace evamx_dense
