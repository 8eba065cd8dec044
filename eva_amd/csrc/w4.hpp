// 4-bit weights with group scales on gfx950: W[n][k] = scale[n][k/G] * (code[n][k] - zero[n][k/G]), codes 0..15, zero 8
// where a matrix has no zero points.
//
// Layout (evamx_w4_pack), per matrix [n_out][n_in]:
//   - codes: tiles of 16 rows of W (the output columns of a product) by 128 k, [n_out/16][n_in/128] tiles of 1 KiB, both
//     counts rounded up. Lane c + 16 g of a wave owns the 16 bytes at 16 (c + 16 g) of a tile: dword j holds column c at
//     k = 32 j + 8 g .. + 7. That is the B operand of v_mfma_f32_16x16x32_f16 (lane c + 16 g: column c, 8 k of the group g):
//     one 16-byte load a lane (1 KiB a wave, contiguous) feeds four matrix instructions with no exchange between lanes.
//   - a dword's nibble i holds k = 2 (i & 3) + (i >> 2) of its 8: nibbles 0 and 4 are a pair of neighbouring k, and so on, so
//     that the pairs come out of the dword by masks alone (w4_operand).
//   - scales (fp16 or bf16) and zero points (bytes): [n_out/16][n_in/512][16 columns][4 k-tiles x 128/G groups], so a lane
//     takes the groups of its column for four k-tiles with one load. Padding columns and k have scale 0 and code 0.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/evamx.h"

namespace evamx {

typedef _Float16 w4_half;
typedef _Float16 w4_half2 __attribute__((ext_vector_type(2)));
typedef _Float16 w4_half8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int W4_TILE_N = 16, W4_TILE_K = 128, W4_TILE_DWORDS = 256;
constexpr int W4_QUAD = 4;                       // k-tiles whose scales lie together

// A stack of matrices as the kernels take it.
struct W4Mat {
    const uint32_t* codes;
    const uint16_t* scales;
    const uint8_t* zeros;                        // NULL: 8 everywhere
    int n_out, n_in, kt, qt, bf16;               // k-tiles, quads of k-tiles, scale type
    size_t tiles, groups;                        // code tiles and scales per matrix
};

__host__ __device__ inline int w4_ceil(int a, int b) { return (a + b - 1) / b; }

inline W4Mat w4_mat(const evamx_w4_weight& w)
{
    W4Mat m;
    m.codes = (const uint32_t*)w.codes;
    m.scales = (const uint16_t*)w.scales;
    m.zeros = (const uint8_t*)w.zeros;
    m.n_out = w.n_out;
    m.n_in = w.n_in;
    m.kt = w4_ceil(w.n_in, W4_TILE_K);
    m.qt = w4_ceil(m.kt, W4_QUAD);
    m.bf16 = w.scale_dtype == EVAMX_DTYPE_BF16;
    m.tiles = (size_t)w4_ceil(w.n_out, W4_TILE_N) * m.kt;
    m.groups = (size_t)w4_ceil(w.n_out, W4_TILE_N) * m.qt * (W4_TILE_N * W4_QUAD * (W4_TILE_K / w.group));
    return m;
}

__device__ __forceinline__ float w4_scale(uint16_t bits, int bf16)
{
    return bf16 ? __builtin_bit_cast(float, (uint32_t)bits << 16) : (float)__builtin_bit_cast(w4_half, bits);
}

// -(1024 + z) and -(64 + z), twice: what takes the offsets of w4_operand's two forms and the zero point off.
struct W4Zero {
    w4_half2 lo, hi;
};

__device__ __forceinline__ W4Zero w4_zero(uint32_t z)
{
    const uint32_t a = 0xe400u | z, b = 0xd400u | (z << 4);
    return {__builtin_bit_cast(w4_half2, a * 0x10001u), __builtin_bit_cast(w4_half2, b * 0x10001u)};
}

// The 8 values code - zero of a dword, exact in fp16: a nibble in the low four bits of a half with the exponent of 1024 is
// 1024 + q, in the next four with the exponent of 64 it is 64 + q (ulp 1/16). 4 v_and_or, 1 shift and 4 packed fp16 adds.
__device__ __forceinline__ w4_half8 w4_operand(uint32_t w, const W4Zero& z)
{
    const uint32_t v = w >> 8;
    const w4_half2 a = __builtin_bit_cast(w4_half2, (w & 0x000f000fu) | 0x64006400u) + z.lo;
    const w4_half2 b = __builtin_bit_cast(w4_half2, (w & 0x00f000f0u) | 0x54005400u) + z.hi;
    const w4_half2 c = __builtin_bit_cast(w4_half2, (v & 0x000f000fu) | 0x64006400u) + z.lo;
    const w4_half2 d = __builtin_bit_cast(w4_half2, (v & 0x00f000f0u) | 0x54005400u) + z.hi;
    return w4_half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The groups of a lane's column for one quad of k-tiles.
template <int SG>
struct W4Groups {
    uint16_t s[W4_QUAD * SG];
    uint8_t z[W4_QUAD * SG];
};

template <int SG, bool ZERO>
__device__ __forceinline__ void w4_load_groups(W4Groups<SG>& g, const W4Mat& m, size_t mat, int nt, int quad, int col)
{
    const size_t at = mat * m.groups + (((size_t)nt * m.qt + quad) * W4_TILE_N + col) * (W4_QUAD * SG);
    __builtin_memcpy(g.s, __builtin_assume_aligned(m.scales + at, 2 * W4_QUAD * SG < 16 ? 2 * W4_QUAD * SG : 16), sizeof g.s);
    if constexpr (ZERO) __builtin_memcpy(g.z, __builtin_assume_aligned(m.zeros + at, W4_QUAD * SG), sizeof g.z);
}

// acc[i] += sum over the k-tiles of the quads q0, q0 + step, .. of a (16 x k) times column tile nt of matrix mat: lane
// c + 16 g holds rows 4 g + i at column c. `a` is the lane's row of activations (row lane & 15 of the block) at its k
// offset 8 (lane >> 4), or NULL for a row that is not there (zeros). Each group's products are summed on the matrix cores
// from zero and then added to the sums times the group's scale, in fp32: neither scale nor code - zero is rounded.
template <int SG, bool ZERO>
__device__ __forceinline__ void w4_accumulate(w4_f32x4& acc, const W4Mat& m, size_t mat, int nt, const w4_half* a, int q0, int step)
{
    const int lane = threadIdx.x & 63;
    const uint32_t* codes = m.codes + (mat * m.tiles + (size_t)nt * m.kt) * W4_TILE_DWORDS + 4 * lane;
    const w4_half8 none = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int q = q0; q < m.qt; q += step) {
        W4Groups<SG> grp;
        w4_load_groups<SG, ZERO>(grp, m, mat, nt, q, lane & 15);
#pragma unroll
        for (int t = 0; t < W4_QUAD; ++t) {
            const int kt = W4_QUAD * q + t;
            if (kt >= m.kt) break;
            const w4_u32x4 w = *(const w4_u32x4*)(codes + (size_t)kt * W4_TILE_DWORDS);
            w4_half8 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = a ? *(const w4_half8*)(a + kt * W4_TILE_K + 32 * j) : none;
            w4_f32x4 part = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s = t * SG + j * SG / 4;
                const W4Zero z = w4_zero(ZERO ? grp.z[s] : 8);
                part = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[j], w4_operand(w[j], z), part, 0, 0, 0);
                if ((j + 1) * SG % 4 == 0) {
                    acc += part * w4_scale(grp.s[s], m.bf16);
                    part = w4_f32x4{0, 0, 0, 0};
                }
            }
        }
    }
}

// A result of x's type, to nearest even; NaN stays.
__device__ __forceinline__ void w4_store(void* y, size_t at, float v, int bf16)
{
    if (bf16) {
        uint32_t b = __builtin_bit_cast(uint32_t, v);
        b = (b & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : b + 0x7fffu + ((b >> 16) & 1);
        ((uint16_t*)y)[at] = (uint16_t)(b >> 16);
    } else {
        ((w4_half*)y)[at] = (w4_half)v;
    }
}

// Exponent that takes a row whose largest finite magnitude has the bits `top` into [2^14, 2^15).
__device__ __forceinline__ int w4_exponent(uint32_t top)
{
    const int e = (int)(top >> 23) - 127 - 14;
    return top == 0 ? 0 : e < -126 ? -126 : e;            // 2^-e stays finite, 2^e normal
}

// f(groups per k-tile, zero points or none) with both as types, for the kernels built for them.
template <class F>
inline void w4_dispatch(const evamx_w4_weight& w, F f)
{
    using std::integral_constant;
    const std::true_type yes;
    const std::false_type no;
    auto pick = [&](auto sg) { if (w.zeros) f(sg, yes); else f(sg, no); };
    if (w.group == 32) pick(integral_constant<int, 4>());
    else if (w.group == 64) pick(integral_constant<int, 2>());
    else pick(integral_constant<int, 1>());
}

// Rows of activations made ready for the products: fp16 [rows][kt * 128] of x * 2^-e, zeros past n_in, and 2^e per row,
// e the exponent that puts the row's largest finite value into [2^14, 2^15). The factor is a power of two, so bf16 values
// down to 2^-28 of the largest are exact in fp16 and none overflows, whatever the row's range; fp32 values (a layer's
// hidden activations) are rounded to fp16's 11 bits. Infinities and NaN stay what they are.
// src_dtype: EVAMX_DTYPE_F16, EVAMX_DTYPE_BF16 or W4_SRC_F32.
constexpr int W4_SRC_F32 = 2;
void w4_launch_rows(const void* src, int src_dtype, size_t src_stride, int rows, int n_in, void* dst, float* scale, hipStream_t stream);

bool w4_weight_ok(const evamx_w4_weight* w, const char* who);

inline size_t w4_align(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace evamx
