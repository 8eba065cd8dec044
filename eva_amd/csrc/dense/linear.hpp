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
    int inter;                   // SwiGLU: n_out / 2, else 0
    int act;
    float limit;
    float* part;                 // [splits][rows][n_out] partial sums, or NULL
    int splits, aligned_y;
};

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

// N (4 or 8) consecutive results at column n of row `row`: v as summed, for SwiGLU the gate's, u the up product's.
template <class T, bool GATED, int N>
__device__ __forceinline__ void finish(const LinearParams& p, int expert, int row, int n, float (&v)[N], float (&u)[N])
{
    constexpr bool BF = std::is_same<T, Bf16>::value;
    const int cols = GATED ? p.inter : p.n_out, have = cols - n;
    if (have <= 0) return;
    auto get = [&](const uint16_t* from, float (&out)[N]) {
        if (have >= N) {
            if constexpr (N == 8) {
                load8(out, from, 8, BF);
            } else {
                const u16x4 x = *(const u16x4_loose*)from;
#pragma unroll
                for (int i = 0; i < N; ++i) out[i] = T::get(x[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = i < have ? T::get(from[i]) : 0.0f;
        }
    };
    float t[N];
    if (p.bias) {
        const uint16_t* b = p.bias + (size_t)expert * p.n_out + n;
        get(b, t);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += t[i];
        if (GATED) {
            get(b + p.inter, t);
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] += t[i];
        }
    }
    if (p.pre) {
        float* at = p.pre + (size_t)row * p.n_out + n;
        store_floats(at, v, have);
        if (GATED) store_floats(at + p.inter, u, have);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = GATED ? swiglu(v[i], u[i], p.limit) : activate(v[i], p.act);
    if (p.residual) {
        get(p.residual + (size_t)row * p.residual_stride + n, t);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += t[i];
    }
    uint16_t* y = p.y + (size_t)row * p.y_stride + n;
    if (have >= N) {
        if constexpr (N == 8) {
            u16x8 o;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = T::put(v[i]);
            *(u16x8_loose*)y = o;
        } else {
            u16x4 o;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = T::put(v[i]);
            *(u16x4_loose*)y = o;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < have) y[i] = T::put(v[i]);
    }
}

int launch_tiles(const LinearParams& p, int dtype, bool transposed, bool loose, hipStream_t s);
int launch_few(const LinearParams& p, int dtype, bool loose, hipStream_t s);
int launch_join(const LinearParams& p, int dtype, hipStream_t s);

}  // namespace evamx_dense
