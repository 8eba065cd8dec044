// Products on 16-bit weights, one matrix for all rows or one for each expert's rows: what their kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../../include/evamx_dense.h"

namespace evamx_dense {

void set_error(const char* fmt, ...);
int launched(const char* what);

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef u16x8 u16x8_loose __attribute__((aligned(2)));      // 16 bytes at any value's address: the hardware takes them, only slower
typedef u16x4 u16x4_loose __attribute__((aligned(2)));

typedef f32x4 f32x4_loose __attribute__((aligned(4)));

// N (4 or 8) floats in a row, or as many as there are.
template <int N>
__device__ __forceinline__ void store_floats(float* p, const float (&v)[N], int have)
{
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if (have >= i + 4) {
            *(f32x4_loose*)(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
#pragma unroll
            for (int j = i; j < i + 3; ++j)
                if (j < have) p[j] = v[j];
        }
    }
}
template <int N>
__device__ __forceinline__ void add_floats(float (&v)[N], const float* p, int have)
{
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if (have >= i + 4) {
            const f32x4 x = *(const f32x4_loose*)(p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] += x[j];
        } else {
#pragma unroll
            for (int j = i; j < i + 3; ++j)
                if (j < have) v[j] += p[j];
        }
    }
}

constexpr int MAX_EXPERTS = 1024, CUS = 256;

struct Bf16 {
    static __device__ __forceinline__ float get(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
    static __device__ __forceinline__ f32x4 mfma(u16x8 a, u16x8 b, f32x4 c)
    {
#ifdef __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
#else
        return c;
#endif
    }
};
struct F16 {
    static __device__ __forceinline__ float get(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ f32x4 mfma(u16x8 a, u16x8 b, f32x4 c)
    {
#ifdef __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#else
        return c;
#endif
    }
};

// Eight values from p on where no row starts at more than a value's address: whole 4-byte words and a shift (a load whose words straddle
// takes about three times as long: 13 rows, 5001 -> 2304, 24 us against 10 for 5000). Reads one value in front of p and two behind the eight.
__device__ __forceinline__ u16x8 load8_shifted(const uint16_t* p)
{
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef u32x4 words __attribute__((aligned(4)));
    const uint32_t* at = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
    const int shift = (int)((uintptr_t)p & 2) * 8;
    const u32x4 v = *(const words*)at;
    const uint32_t end = at[4];
    u32x4 o;
    o[0] = __builtin_amdgcn_alignbit(v[1], v[0], shift);
    o[1] = __builtin_amdgcn_alignbit(v[2], v[1], shift);
    o[2] = __builtin_amdgcn_alignbit(v[3], v[2], shift);
    o[3] = __builtin_amdgcn_alignbit(end, v[3], shift);
    return __builtin_bit_cast(u16x8, o);
}

// ---- activations ------------------------------------------------------------------------------

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

// The normal distribution function: its smaller side is erfc(z) / 2 = t 2^(P(t) - z^2 / ln 2) at z = |v| / sqrt(2), t = 1 / (1 + 0.4 z),
// with P fitted here at the Chebyshev points of z = 0 .. 10, to 1.1e-7 of erfc; in these 32 bits 8e-7 of the value for |v| < 3, 8e-6 for 13.
// (0.5 (1 + erff) loses the lower side, and costs as much as a product of 64 values: 300 rows of 2048 -> 7168 with bias and residual
// 46 us instead of 39.)
__device__ __forceinline__ float normal(float v)
{
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.282842712f, fabsf(v), 1.0f));
    float e = -0.306892693f;
    e = __builtin_fmaf(e, t, 1.37083006f);
    e = __builtin_fmaf(e, t, -2.22021937f);
    e = __builtin_fmaf(e, t, 1.52885067f);
    e = __builtin_fmaf(e, t, -0.699879766f);
    e = __builtin_fmaf(e, t, 0.458745331f);
    e = __builtin_fmaf(e, t, 0.570344865f);
    e = __builtin_fmaf(e, t, 1.44602776f);
    e = __builtin_fmaf(e, t, -3.14780688f);
    const float low = t * __builtin_amdgcn_exp2f(__builtin_fmaf(-0.72134752f * v, v, e));
    return v > 0 ? 1.0f - low : low;
}

// Clamps that leave a NaN as it is.
__device__ __forceinline__ float at_most(float v, float m) { return v > m ? m : v; }
__device__ __forceinline__ float within(float v, float m) { return v > m ? m : v < -m ? -m : v; }

__device__ __forceinline__ float swiglu(float gate, float up, float limit)
{
    const float a = gate * sigmoid(gate);
    return limit > 0 ? at_most(a, limit) * within(up, limit) : a * up;
}

template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    if (act == EVAMX_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * sigmoid(v[i]);
    } else if (act == EVAMX_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * normal(v[i]);
    } else if (act == EVAMX_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0 ? 0.0f : v[i];
    }
}

// Its derivative.
__device__ __forceinline__ float slope(float v, int act)
{
    if (act == EVAMX_ACT_SILU) {
        const float s = sigmoid(v);
        return s * (1.0f + v * (1.0f - s));
    }
    if (act == EVAMX_ACT_GELU) return normal(v) + v * 0.39894228f * __expf(-0.5f * v * v);
    return v > 0 ? 1.0f : v == v ? 0.0f : v;                     // ReLU; a NaN stays one
}

// ---- which rows a workgroup takes ---------------------------------------------------------------

// Rows of expert e are [starts[e], starts[e + 1]), cut to the rows there are, whatever the table holds; without a table all rows
// are one expert's.
struct Groups {
    static constexpr int ALL = 1 << 30;
    const int32_t* starts;
    int experts, rows;
    int above = 0, upto = ALL;    // with a table: the experts of above + 1 to upto rows, others have none

    __device__ __forceinline__ int start(int e) const
    {
        const int v = starts[e];
        return v < 0 ? 0 : v > rows ? rows : v;
    }
    __device__ __forceinline__ int end() const { return starts ? start(experts) : rows; }
};

struct Tile {
    int expert, row, have, col;   // rows row .. row + have - 1 (of a tile of at most TQ), column tile col
};

// The work's tiles: row tiles of TQ of each expert by cols column tiles. They are numbered so that consecutive workgroups, which go to
// the eight XCDs in turn, give each XCD a contiguous run of them: expert by expert, within one eight row tiles by all columns at a
// time, so that neighbours share their rows and weights in the L2. All threads call init() and find(); s: 2 + THREADS / 64 ints of LDS
// for them alone.
template <int THREADS, int TQ>
struct Tiles {
    static constexpr int PER = (MAX_EXPERTS + THREADS - 1) / THREADS;
    Groups g;
    int* s;
    int cols, all, each;          // tiles in all, and of an XCD
    int upto, mine, per, count[PER];   // a thread's experts: row tiles up to and with them, theirs, and their rows

    __device__ __forceinline__ void init(const Groups& groups, int columns, int* scratch)
    {
        g = groups; cols = columns; s = scratch;
        int total;
        if (g.starts) {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            per = (g.experts + THREADS - 1) / THREADS;
            mine = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = (int)threadIdx.x * per + i;
                count[i] = i < per && e < g.experts ? g.start(e + 1) - g.start(e) : 0;
                if (count[i] <= g.above || count[i] > g.upto) count[i] = 0;
                mine += (count[i] + TQ - 1) / TQ;
            }
            upto = mine;
            for (int d = 1; d < 64; d <<= 1) {
                const int n = __shfl_up(upto, d);
                if (lane >= d) upto += n;
            }
            if (lane == 63) s[2 + wave] = upto;
            __syncthreads();
            total = 0;
            for (int w = 0; w < THREADS / 64; ++w) {
                if (w < wave) upto += s[2 + w];
                total += s[2 + w];
            }
        } else {
            total = (g.rows + TQ - 1) / TQ;
        }
        all = __builtin_amdgcn_readfirstlane(total * cols);
        each = (all + 7) / 8;
    }
    // Work item u < 8 * each; false: it has no tile.
    __device__ __forceinline__ bool find(int u, Tile& tile)
    {
        int t = (u & 7) * each + u / 8, e = 0, begin = 0, rows = g.rows;
        if (u / 8 >= each || t >= all) return false;
        if (g.starts) {
            const int row_tile = t / cols;
            __syncthreads();                                           // the last call's answer has been read
            if (row_tile >= upto - mine && row_tile < upto) {          // one thread's
                int before = upto - mine;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int n = (count[i] + TQ - 1) / TQ;
                    if (row_tile >= before && row_tile < before + n) {
                        s[0] = (int)threadIdx.x * per + i;
                        s[1] = before;
                    }
                    before += n;
                }
            }
            __syncthreads();
            e = __builtin_amdgcn_readfirstlane(s[0]);
            t -= __builtin_amdgcn_readfirstlane(s[1]) * cols;
            begin = g.start(e);
            rows = g.start(e + 1) - begin;
        }
        const int row_tiles = (rows + TQ - 1) / TQ, band = t / (8 * cols), in_band = t - band * 8 * cols;
        const int deep = row_tiles - 8 * band < 8 ? row_tiles - 8 * band : 8;
        const int r = TQ * (8 * band + in_band % deep);
        tile.expert = e;
        tile.row = begin + r;
        tile.have = rows - r < TQ ? rows - r : TQ;
        tile.col = in_band / deep;
        return true;
    }
};

// 16 bytes of a result. STREAM: not to stay in the L2, for results of more than the last-level cache holds, and what nothing reads.
template <bool STREAM>
__device__ __forceinline__ void store16(uint16_t* p, u16x8 v)
{
    if constexpr (STREAM) __builtin_nontemporal_store(v, (u16x8_loose*)p);
    else *(u16x8_loose*)p = v;
}
constexpr int64_t CACHE = 256 << 20;

// Zeros in rows [from, rows) of out, which nothing needs: those of workgroup b of n (4096 tokens at an eighth of the experts, 8 slots,
// seven eighths of the rows: y 444 us against 461 with plain stores, x's gradient 497 against 514).
__device__ __forceinline__ void zero_rows(uint16_t* out, size_t stride, int cols, int64_t from, int64_t rows, int b, int n)
{
    for (int64_t r = from + b; r < rows; r += n) {
        uint16_t* at = out + (size_t)r * stride;
        for (int c = threadIdx.x * 8; c < cols; c += blockDim.x * 8) {
            if (c + 8 <= cols) {
                store16<true>(at + c, (u16x8)(uint16_t)0);
            } else {
                for (int i = c; i < cols; ++i) at[i] = 0;
            }
        }
    }
}

static inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
// Row tiles that the rows can make at most.
static inline int64_t most_row_tiles(const Groups& g, int tq)
{
    if (!g.starts) return ceil_div(g.rows, tq);
    const int64_t most = g.rows / (g.above + 1), experts = most < g.experts ? most : g.experts;    // that have rows
    return (g.upto < tq ? 0 : g.rows / tq) + experts;
}

}  // namespace evamx_dense
