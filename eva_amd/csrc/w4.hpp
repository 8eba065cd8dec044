// 4-bit weights with group scales on gfx950: W[n][k] = scale[n][k/G] * (code[n][k] - zero[n][k/G]), codes 0..15, zero
// points 0..31, or 8 where a matrix has none.
//
// Layout (evamx_w4_pack), per matrix [n_out][n_in]:
//   - codes: tiles of 16 rows of W (the output columns of a product) by 128 k, [n_out/16][n_in/128] tiles of 1 KiB, both
//     counts rounded up. Lane c + 16 g of a wave owns the 16 bytes at 16 (c + 16 g) of a tile: dword j holds column c at
//     k = 32 j + 8 g .. + 7. That is the B operand of v_mfma_f32_16x16x32_f16 (lane c + 16 g: column c, 8 k of the group g):
//     one 16-byte load a lane (1 KiB a wave, contiguous) feeds four matrix instructions with no exchange between lanes.
//   - a dword's nibble i holds k = 2 (i & 3) + (i >> 2) of its 8: nibbles 0 and 4 are a pair of neighbouring k, and so on, so
//     that the pairs come out of the dword by masks alone (w4_operand).
//   - scales (fp16 or bf16) and zero points (bytes): [n_out/16][n_in/128][16 columns][128/G groups], so a lane takes the
//     groups of its column in a k-tile with one load. Padding columns and k have scale 0 and code 0.
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
constexpr uint32_t W4_ZERO_MAX = 31;         // zero points are the low five bits of their bytes, here and in evamx_w4_dequant

// A stack of matrices as the kernels take it.
struct W4Mat {
    const uint32_t* codes;
    const uint16_t* scales;
    const uint8_t* zeros;                        // NULL: 8 everywhere
    int n_out, n_in, nt, kt, bf16;               // column tiles, k-tiles, scale type
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
    m.nt = w4_ceil(w.n_out, W4_TILE_N);
    m.kt = w4_ceil(w.n_in, W4_TILE_K);
    m.bf16 = w.scale_dtype == EVAMX_DTYPE_BF16;
    m.tiles = (size_t)m.nt * m.kt;
    m.groups = m.tiles * (W4_TILE_N * (W4_TILE_K / w.group));
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

// The masks and exponents of w4_operand, where one instruction can take a mask and an exponent: masks in scalar, exponents in
// vector registers. As literals they would cost an AND and an OR (13 instead of 9 instructions a dword).
struct W4Consts {
    uint32_t m0, m1, e0, e1;
    __device__ __forceinline__ W4Consts() : m0(0x000f000fu), m1(0x00f000f0u), e0(0x64006400u), e1(0x54005400u)
    {
        asm volatile("" : "+s"(m0), "+s"(m1), "+v"(e0), "+v"(e1));
    }
};

// The 8 values code - zero of a dword, exact in fp16: a nibble in the low four bits of a half with the exponent of 1024 is
// 1024 + q, in the next four with the exponent of 64 it is 64 + q (ulp 1/16). 4 v_and_or, 1 shift and 4 packed fp16 adds.
__device__ __forceinline__ w4_half8 w4_operand(uint32_t w, const W4Zero& z, const W4Consts& k)
{
    const uint32_t v = w >> 8;
    const w4_half2 a = __builtin_bit_cast(w4_half2, (w & k.m0) | k.e0) + z.lo;
    const w4_half2 b = __builtin_bit_cast(w4_half2, (w & k.m1) | k.e1) + z.hi;
    const w4_half2 c = __builtin_bit_cast(w4_half2, (v & k.m0) | k.e0) + z.lo;
    const w4_half2 d = __builtin_bit_cast(w4_half2, (v & k.m1) | k.e1) + z.hi;
    return w4_half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// One column tile of one matrix, its k-tiles up to an end: descriptors of wave-uniform bases (in scalar registers). Loads past
// the end return zeros and touch no memory, so a wave can request tiles ahead without a test.
struct W4Stream {
    __amdgpu_buffer_rsrc_t codes, scales, zeros;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_rsrc(const void* base, uint32_t bytes)
{
    const uint64_t v = (uint64_t)(uintptr_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)(((uint64_t)hi << 32) | lo), (short)0, __builtin_amdgcn_readfirstlane(bytes),
                                             0x00027000);
}

template <int SG, bool ZERO>
__device__ __forceinline__ W4Stream w4_stream(const W4Mat& m, size_t mat, int nt, int kt_end)
{
    const size_t tile = (size_t)nt * m.kt, grp = mat * m.groups + tile * (W4_TILE_N * SG);
    W4Stream st;
    st.codes = w4_rsrc(m.codes + (mat * m.tiles + tile) * W4_TILE_DWORDS, (uint32_t)kt_end * (W4_TILE_DWORDS * 4));
    st.scales = w4_rsrc(m.scales + grp, (uint32_t)kt_end * (W4_TILE_N * SG * 2));
    if constexpr (ZERO) st.zeros = w4_rsrc(m.zeros + grp, (uint32_t)kt_end * (W4_TILE_N * SG));
    return st;
}

// A lane's share of one tile, as loaded.
template <int SG>
struct W4Raw {
    w4_u32x4 c;
    uint32_t s[SG == 4 ? 2 : 1], z;
};

template <int SG, bool ZERO>
__device__ __forceinline__ void w4_load(W4Raw<SG>& r, const W4Stream& st, int kt)
{
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const int lane = threadIdx.x & 63, at = kt * W4_TILE_N + (lane & 15);
    r.c = __builtin_bit_cast(w4_u32x4, __builtin_amdgcn_raw_buffer_load_b128(st.codes, kt * (W4_TILE_DWORDS * 4) + lane * 16, 0, 0));
    if constexpr (SG == 1) {
        r.s[0] = __builtin_amdgcn_raw_buffer_load_b16(st.scales, at * 2, 0, 0);
        if constexpr (ZERO) r.z = __builtin_amdgcn_raw_buffer_load_b8(st.zeros, at, 0, 0);
    } else if constexpr (SG == 2) {
        r.s[0] = __builtin_amdgcn_raw_buffer_load_b32(st.scales, at * 4, 0, 0);
        if constexpr (ZERO) r.z = __builtin_amdgcn_raw_buffer_load_b16(st.zeros, at * 2, 0, 0);
    } else {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(st.scales, at * 8, 0, 0));
        r.s[0] = v.x;
        r.s[1] = v.y;
        if constexpr (ZERO) r.z = __builtin_amdgcn_raw_buffer_load_b32(st.zeros, at * 4, 0, 0);
    }
}

// acc[mb] += the products of MB blocks of 16 rows with one tile: lane c + 16 g holds rows 4 g + i at column c, of which the
// first NR are wanted. A group's products are summed on the matrix cores from zero and then added times the group's scale in
// fp32: neither scale nor code - zero is rounded. HL: the rows' values are the sums of two fp16 halves, x and lo.
template <int SG, bool ZERO, int MB, int NR, bool HL>
__device__ __forceinline__ void w4_tile(w4_f32x4 (&acc)[MB], const W4Raw<SG>& r, const w4_half8 (&x)[MB][4], const w4_half8 (&lo)[MB][4], int bf16,
                                        const W4Consts& consts)
{
#pragma unroll
    for (int g = 0; g < SG; ++g) {
        const W4Zero z = w4_zero(ZERO ? (r.z >> (8 * g)) & W4_ZERO_MAX : 8);
        w4_f32x4 part[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) part[mb] = w4_f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = g * (4 / SG); j < (g + 1) * (4 / SG); ++j) {
            const w4_half8 b = w4_operand(r.c[j], z, consts);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                part[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[mb][j], b, part[mb], 0, 0, 0);
                if constexpr (HL) part[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[mb][j], b, part[mb], 0, 0, 0);
            }
        }
        const float s = w4_scale((uint16_t)(r.s[g >> 1] >> (16 * (g & 1))), bf16);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int i = 0; i < NR; ++i) acc[mb][i] = __builtin_fmaf(part[mb][i], s, acc[mb][i]);
    }
}

// The k-tiles of a row are cut into parts, a wave each; a result is the sum of its parts in order. The cut depends on the
// matrix alone, so up to 16 rows a row has the same bits in every batch.
__host__ __device__ inline int w4_part_begin(int kt, int parts, int i) { return (int)((long)kt * i / parts); }

// Parts of a single matrix: enough waves to keep the memory busy, few enough that each has several tiles in flight; twice as
// many where the columns alone make few workgroups (5001 -> 2303 at 13 rows: 11.9 us with 8, 12.3 with 4).
inline int w4_parts(int kt, int nt) { return kt >= 32 && nt < 512 ? 8 : kt >= 8 ? 4 : kt >= 2 ? 2 : 1; }
constexpr int W4_MAX_PARTS = 8;

// acc[b][mb] += rows times the k-tiles [k0, k1) of NB streams, RING tiles of each in flight. `rows(d, kt, x, lo)` gives the lane's
// activations of a tile at the time its products are due; `ahead(d, kt)` is called with each request for tile kt into place d of
// the ring, `begin()` once the first are under way.
template <int RING, int SG, bool ZERO, int NB, int MB, int NR, bool HL, class Ahead, class Rows, class Begin>
__device__ __forceinline__ void w4_run(w4_f32x4 (&acc)[NB][MB], const W4Stream (&st)[NB], int k0, int k1, int bf16, Ahead&& ahead, Rows&& rows,
                                       Begin&& begin)
{
    W4Raw<SG> ring[RING][NB];
    const W4Consts consts;
    k0 = __builtin_amdgcn_readfirstlane(k0);
    k1 = __builtin_amdgcn_readfirstlane(k1);
#pragma unroll
    for (int d = 0; d < RING; ++d) {
#pragma unroll
        for (int b = 0; b < NB; ++b) w4_load<SG, ZERO>(ring[d][b], st[b], k0 + d);
        ahead(d, k0 + d);
    }
    begin();
    for (int kt = k0; kt < k1; kt += RING) {
#pragma unroll
        for (int d = 0; d < RING; ++d) {
            if (kt + d < k1) {
                w4_half8 x[MB][4], lo[MB][4];
                rows(d, kt + d, x, lo);
#pragma unroll
                for (int b = 0; b < NB; ++b) w4_tile<SG, ZERO, MB, NR, HL>(acc[b], ring[d][b], x, lo, bf16, consts);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) w4_load<SG, ZERO>(ring[d][b], st[b], kt + d + RING);
            ahead(d, kt + d + RING);
        }
    }
}

// Activations in global memory, made ready by w4_launch_rows: requested with the tiles they multiply (from a descriptor, as
// the weights: plain loads would be sunk to their use). at[mb]: byte offset of the lane's row at its k offset 8 (lane >> 4);
// a low half lies lo_off bytes behind. Offsets are below 2^32 (the entry points see to it).
template <int MB, bool HL>
struct W4GlobalRows {
    __amdgpu_buffer_rsrc_t src;
    uint32_t at[MB], lo_off;
    w4_half8 buf[MB][4], low[HL ? MB : 1][4];

    __device__ __forceinline__ void request(int kt)
    {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t o = at[mb] + (uint32_t)kt * (W4_TILE_K * 2) + 64 * j;
                buf[mb][j] = __builtin_bit_cast(w4_half8, __builtin_amdgcn_raw_buffer_load_b128(src, o, 0, 0));
                if constexpr (HL) low[mb][j] = __builtin_bit_cast(w4_half8, __builtin_amdgcn_raw_buffer_load_b128(src, o + lo_off, 0, 0));
            }
    }

    __device__ __forceinline__ void take(w4_half8 (&x)[MB][4], w4_half8 (&lo)[MB][4]) const
    {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[mb][j] = buf[mb][j];
                if constexpr (HL) lo[mb][j] = low[mb][j];
            }
    }
};

// Exponent that takes a row whose largest finite magnitude has the bits `top` into [2^14, 2^15).
__device__ __forceinline__ int w4_exponent(uint32_t top)
{
    const int e = (int)(top >> 23) - 127 - 14;
    return top == 0 ? 0 : e < -126 ? -126 : e;            // 2^-e stays finite, 2^e normal
}

// A row of activations made ready by THREADS threads (a wave or a workgroup) for w4_tile: load() requests it, 8 values a thread
// and chunk, finish() writes fp16 values times 2^-e and returns 2^e, e the exponent that takes the row's largest finite
// magnitude into [2^14, 2^15) (0 for fp16 rows, which need none). The factor is a power of two, so bf16 values down to 2^-28
// of the largest are exact and none overflows. Of fp32 rows (hidden activations) the values are fp16's 11 bits and, with HL, what
// that leaves in a second half lo_off values on. Zeros from n_in to n_pad. Rows longer than NC chunks are read twice.
constexpr int W4_SRC_F32 = 2;

template <int SRC, int THREADS, bool HL>
struct W4ReadyRow {
    static constexpr int NC = 4;
    const char* row;
    int n_in, n_pad;
    bool aligned;                                // the row starts at a 16-byte address
    int tid;
    float v[NC][8];

    __device__ __forceinline__ void load8(int k, float (&o)[8]) const
    {
        constexpr int SIZE = SRC == W4_SRC_F32 ? 4 : 2;
        if (aligned && k + 8 <= n_in) {
            const w4_u32x4* src = (const w4_u32x4*)(row + (size_t)k * SIZE);
            const w4_u32x4 a = src[0];
            if constexpr (SRC == W4_SRC_F32) {
                const w4_u32x4 b = src[1];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = __builtin_bit_cast(float, e < 4 ? a[e & 3] : b[e & 3]);
            } else if constexpr (SRC == EVAMX_DTYPE_BF16) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = __builtin_bit_cast(float, e & 1 ? a[e >> 1] & 0xffff0000u : a[e >> 1] << 16);
            } else {
                const w4_half8 h = __builtin_bit_cast(w4_half8, a);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (float)h[e];
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[e] = 0.0f;
            if (k + e >= n_in) continue;
            if constexpr (SRC == W4_SRC_F32) o[e] = ((const float*)row)[k + e];
            else if constexpr (SRC == EVAMX_DTYPE_BF16) o[e] = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[k + e] << 16);
            else o[e] = (float)((const w4_half*)row)[k + e];
        }
    }

    __device__ __forceinline__ void load()
    {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = 8 * (c * THREADS + tid);
            if (k < n_pad) load8(k, v[c]);
        }
    }

    static __device__ __forceinline__ uint32_t most(const float (&o)[8], uint32_t top)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = __builtin_bit_cast(uint32_t, o[e]) & 0x7fffffffu;
            top = b < 0x7f800000u && b > top ? b : top;
        }
        return top;
    }

    static __device__ __forceinline__ void put(w4_half* dst, int lo_off, const float (&o)[8], float down)
    {
        w4_half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = o[e] * down;
            h[e] = (w4_half)x;
            if constexpr (HL) {
                const float left = x - (float)h[e];
                l[e] = (w4_half)(left == left ? left : 0.0f);    // of an infinity nothing is left
            }
        }
        *(w4_half8*)dst = h;
        if constexpr (HL) *(w4_half8*)(dst + lo_off) = l;
    }

    // part: LDS, one word a wave (unused by a single wave)
    __device__ __forceinline__ float finish(w4_half* dst, int lo_off, uint32_t* part) const
    {
        int e = 0;
        if constexpr (SRC != EVAMX_DTYPE_F16) {
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (8 * (c * THREADS + tid) < n_pad) top = most(v[c], top);
            for (int k = 8 * (NC * THREADS + tid); k < n_pad; k += 8 * THREADS) {
                float o[8];
                load8(k, o);
                top = most(o, top);
            }
            for (int s = 32; s; s >>= 1) {
                const uint32_t o = (uint32_t)__shfl_xor((int)top, s);
                top = o > top ? o : top;
            }
            if constexpr (THREADS > 64) {
                if ((tid & 63) == 0) part[tid >> 6] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < THREADS / 64; ++w) top = part[w] > top ? part[w] : top;
            }
            e = w4_exponent(top);
        }
        const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = 8 * (c * THREADS + tid);
            if (k < n_pad) put(dst + k, lo_off, v[c], down);
        }
        for (int k = 8 * (NC * THREADS + tid); k < n_pad; k += 8 * THREADS) {
            float o[8];
            load8(k, o);
            put(dst + k, lo_off, o, down);
        }
        return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
    }
};

// Up to four rows of x, made ready in the workgroup's LDS (as w4_launch_rows does in memory) while the first weights are on
// their way: load() requests them, finish() scales and stores them. Rows lie W4_STAGE_PAD halves apart beyond their length,
// so that the four rows a wave reads at once start in different banks.
constexpr int W4_STAGE_ROWS = 4, W4_STAGE_CHUNKS = 8, W4_STAGE_PAD = 32;

inline size_t w4_stage_bytes(int rows, int kt) { return (size_t)rows * (kt * W4_TILE_K + W4_STAGE_PAD) * 2; }
// Whether `rows` rows of kt k-tiles can be staged by a workgroup of `parts` waves.
inline bool w4_stage_fits(int rows, int kt, int parts)
{
    return rows <= W4_STAGE_ROWS && (long)rows * kt * (W4_TILE_K / 8) <= (long)W4_STAGE_CHUNKS * 64 * parts &&
           w4_stage_bytes(rows, kt) <= 58 * 1024;            // two workgroups a CU
}

struct W4Stage {
    const uint16_t* x;
    size_t stride;
    int rows, n_in, kt, bf16, aligned;           // aligned: rows start at 16-byte addresses
    w4_u32x4 c[W4_STAGE_CHUNKS];

    __device__ __forceinline__ void load()
    {
        const int per = kt * (W4_TILE_K / 8), total = rows * per, n = blockDim.x;
#pragma unroll
        for (int i = 0; i < W4_STAGE_CHUNKS; ++i) {
            c[i] = w4_u32x4{0, 0, 0, 0};
            const int ch = threadIdx.x + i * n;
            if (ch >= total) continue;
            const int r = ch / per, k = (ch - r * per) * 8;
            const uint16_t* src = x + r * stride + k;
            if (aligned && k + 8 <= n_in) {
                c[i] = *(const w4_u32x4*)src;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + e < n_in) c[i][e >> 1] |= (uint32_t)src[e] << (16 * (e & 1));
            }
        }
    }

    // dst: LDS rows; top: LDS [W4_MAX_PARTS][4]; scale: LDS [4], the rows' factors
    __device__ __forceinline__ void finish(w4_half* dst, uint32_t (*top)[4], float* scale)
    {
        const int per = kt * (W4_TILE_K / 8), total = rows * per, n = blockDim.x, ld = kt * W4_TILE_K + W4_STAGE_PAD;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        int e[W4_STAGE_ROWS] = {0, 0, 0, 0};
        if (bf16) {
            uint32_t m[W4_STAGE_ROWS] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < W4_STAGE_CHUNKS; ++i) {
                const int ch = threadIdx.x + i * n, r = ch / per;
                if (ch >= total) continue;
                uint32_t v = 0;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t a = c[i][d] & 0x7fffu, b = (c[i][d] >> 16) & 0x7fffu;
                    v = a < 0x7f80u && a > v ? a : v;
                    v = b < 0x7f80u && b > v ? b : v;
                }
#pragma unroll
                for (int q = 0; q < W4_STAGE_ROWS; ++q) m[q] = r == q && v > m[q] ? v : m[q];
            }
#pragma unroll
            for (int q = 0; q < W4_STAGE_ROWS; ++q) {
                if (q >= rows) break;
                for (int s = 32; s; s >>= 1) {
                    const uint32_t o = (uint32_t)__shfl_xor((int)m[q], s);
                    m[q] = o > m[q] ? o : m[q];
                }
                if (lane == 0) top[wave][q] = m[q];
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < W4_STAGE_ROWS; ++q) {
                if (q >= rows) break;
                uint32_t t = 0;
                for (int w = 0; w < n >> 6; ++w) t = top[w][q] > t ? top[w][q] : t;
                e[q] = w4_exponent(t << 16);
            }
        }
        if (threadIdx.x < rows) scale[threadIdx.x] = __builtin_bit_cast(float, (uint32_t)(127 + e[threadIdx.x & 3]) << 23);
#pragma unroll
        for (int i = 0; i < W4_STAGE_CHUNKS; ++i) {
            const int ch = threadIdx.x + i * n, r = ch / per;
            if (ch >= total) continue;
            w4_u32x4 v = c[i];
            if (bf16) {
                const int er = r == 0 ? e[0] : r == 1 ? e[1] : r == 2 ? e[2] : e[3];
                const float down = __builtin_bit_cast(float, (uint32_t)(127 - er) << 23);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const w4_half2 h = {(w4_half)(__builtin_bit_cast(float, v[d] << 16) * down),
                                        (w4_half)(__builtin_bit_cast(float, v[d] & 0xffff0000u) * down)};
                    v[d] = __builtin_bit_cast(uint32_t, h);
                }
            }
            *(w4_u32x4*)(dst + r * ld + (ch - r * per) * 8) = v;
        }
        __syncthreads();
    }
};

// A result of x's type, to nearest even; NaN stays.
__device__ __forceinline__ uint16_t w4_bits(float v, int bf16)
{
    return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (w4_half)v);
}

__device__ __forceinline__ void w4_store(void* y, size_t at, float v, int bf16) { ((uint16_t*)y)[at] = w4_bits(v, bf16); }

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

// Rows of x made ready in memory (W4ReadyRow): fp16 [rows][kt * 128] and a factor per row.
void w4_launch_rows(const void* src, int src_dtype, size_t src_stride, int rows, int n_in, void* dst, float* scale, hipStream_t stream);

// Rows that are used as they lie: fp16, whole tiles, at 16-byte addresses.
inline bool w4_rows_ready(const void* x, int x_dtype, int64_t x_stride, int n_in)
{
    return x_dtype == EVAMX_DTYPE_F16 && n_in % W4_TILE_K == 0 && x_stride == n_in && ((uintptr_t)x & 15) == 0;
}

bool w4_weight_ok(const evamx_w4_weight* w, const char* who);

inline size_t w4_align(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace evamx
