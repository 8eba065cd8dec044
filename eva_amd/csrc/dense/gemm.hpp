// The tiles of the larger products: acc[p][q] += sum_k P[p][k] Q[q][k] on v_mfma_f32_16x16x32.
//
// p runs along a row of the result (so that a lane ends up with four values in a row), q over its rows. A matrix comes either
// with k along its rows in memory, or (TR) with k over its rows: then LDS holds it as it lies in memory and ds_read_b64_tr_b16
// turns it on the way to the registers. k-tiles of 64 come to LDS directly, into two or three places in turn.
//
// 256 by 256 by 64: 2048 cycles of matrix instructions a CU beside 1536 of LDS reads and 512 of its loads. 8192 rows of 7168 -> 4096 in
// bf16: 365 us, 1320 TFLOP/s (x's gradient 397, w's 383; a large library product 1605): the operands' way from memory, a k-tile ahead,
// and the clock under such loads bound it. 4096^3: 100 us, 1370 TFLOP/s.
#pragma once
#include "dense.hpp"

namespace evamx_dense {

constexpr int TILE_K = 64;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes)
{
    const uint64_t v = (uint64_t)(uintptr_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)(((uint64_t)hi << 32) | lo), (short)0, __builtin_amdgcn_readfirstlane(bytes),
                                             0x00027000);
}

// The rows that one turning read takes together (four of every eight, of sixteen) in eight places.
__device__ __forceinline__ int turn(int row) { return (row & 3) | (row >> 1 & 4); }

// One matrix of a workgroup's product: N values of p or q, by k.
//   k along the rows:  value n is row map(n) of base, cut to `rows` rows, of `len` = K values.
//   TR:                k is the row, cut to `rows` = K rows; value n is column n of base, cut to `len` columns.
// Addresses and lengths are multiples of 16 bytes (what comes otherwise is copied first).
// In LDS in chunks of 16 bytes, in the order in which the direct loads write them; the chunks of a row are swapped by the row's low
// bits (in the addresses that are loaded), so that what an instruction reads together lies in different banks.
template <bool TR, int N, int WAVES>
struct Side {
    static constexpr int BYTES = N * TILE_K * 2, LOADS = BYTES / 1024 / WAVES, ROW_CHUNKS = TR ? N / 8 : TILE_K / 8;
    static_assert(LOADS >= 1 && LOADS * WAVES * 1024 == BYTES);
    const uint16_t* base;
    size_t stride;
    int rows, len;
    uint32_t at[LOADS];           // byte offsets of a lane's chunks
    __amdgpu_buffer_rsrc_t all;   // the whole of the matrix with k along its rows

    static __device__ __forceinline__ int swap(int row) { return TR ? turn(row) * 2 : row & 7; }

    template <class Map>
    __device__ __forceinline__ void init(const uint16_t* b, size_t s, int r, int l, Map map)
    {
        base = b; stride = s; rows = r; len = l;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int slot = (i * WAVES + wave) * 64 + lane, row = slot / ROW_CHUNKS, chunk = (slot % ROW_CHUNKS) ^ swap(row);
            const int from = TR ? row : map(row);
            at[i] = (uint32_t)from * (uint32_t)stride * 2 + chunk * 16;
        }
        if constexpr (!TR) all = buffer(base, rows <= 0 ? 0u : (uint32_t)((rows - 1) * stride + len) * 2);
    }
    // k-tiles before this one end within the rows (TR: a descriptor a k-tile sees to that)
    __device__ __forceinline__ int whole() const { return TR ? 1 << 30 : len / TILE_K; }
    // k-tile kt to LDS at `to`. Rows, columns and k that are not there become zeros; with TR, columns behind the last may hold the
    // next row's values, which end in results that are not stored.
    template <bool WHOLE>         // the k-tile ends within the rows
    __device__ __forceinline__ void bring(char* to, int kt) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k0 = kt * TILE_K;
        if constexpr (TR) {
            const int left = rows - k0 < TILE_K ? rows - k0 : TILE_K;
            const __amdgpu_buffer_rsrc_t src = buffer(base + (size_t)k0 * stride, left <= 0 ? 0u : (uint32_t)((left - 1) * stride + len) * 2);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)(to + (i * WAVES + wave) * 1024), 16, at[i],
                                                         0, 0, 0);
        } else {
            const int left = len - k0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int chunk = ((i * WAVES + wave) * 64 + lane) % ROW_CHUNKS ^ swap(((i * WAVES + wave) * 64 + lane) / ROW_CHUNKS);
                // chunks behind the row's end: no address
                const uint32_t from = WHOLE ? at[i] : chunk * 8 < left ? at[i] : 0xfffffff0u - (uint32_t)k0 * 2;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(all, (__attribute__((address_space(3))) void*)(to + (i * WAVES + wave) * 1024), 16, from,
                                                         k0 * 2, 0, 0);
            }
        }
#endif
    }
};

// Four rows of 16 values of LDS, of which lane l of 16 names the four values 4 (l % 4) of row l / 4, to four rows' values of
// column l. restrict tells the compiler's count of open loads that what is under way to LDS goes elsewhere; without it each read
// waits for all of them (x's gradient of 8192 rows, 4096 -> 7168: 529 us).
__device__ __forceinline__ s16x4 turned(const char* __restrict__ p)
{
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
#else
    return s16x4{};
#endif
}

// What a lane of a wave reads of a side: BLOCKS blocks of 16 values from block `first` on, lane c + 16 g the k 8 g .. 8 g + 7 of
// each 32.
template <bool TR, int N, int BLOCKS>
struct Reader {
    static constexpr int BASES = TR ? BLOCKS : 2;
    uint32_t at[BASES];

    // step: the half of a k-tile that read()'s step 0 is
    __device__ __forceinline__ void init(int first, int step)
    {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        if constexpr (!TR) {
            at[0] = (16 * first + c) * (TILE_K * 2) + (((g + 4 * step) ^ (c & 7)) * 16);
            at[1] = at[0] ^ 64;
        } else {
            const int row = 32 * step + 8 * g + (c >> 2);
#pragma unroll
            for (int j = 0; j < BASES; ++j) at[j] = row * (N * 2) + ((first + j) ^ turn(row)) * 32 + 8 * (c & 3);
        }
    }
    __device__ __forceinline__ u16x8 read(const char* lds, int step, int b) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        if constexpr (!TR) {
            return *(const u16x8*)(lds + at[step] + b * (16 * TILE_K * 2));
        } else {
            const char* p = lds + at[b] + step * (32 * N * 2);
            return __builtin_bit_cast(u16x8, __builtin_shufflevector(turned(p), turned(p + 4 * N * 2), 0, 1, 2, 3, 4, 5, 6, 7));
        }
#else
        return u16x8{};
#endif
    }
};

template <int N>
__device__ __forceinline__ void wait_loads()                            // s_waitcnt vmcnt(N)
{
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | 15 << 8 | (N >> 4) << 14);
}
__device__ __forceinline__ void arrive()                                // all waves are here, and their LDS accesses are done
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A wave's place in LDS for results on their way out: 64 rows, OUT_ROW floats apart (rows_of).
constexpr int OUT_ROW = 68, OUT_BYTES = 64 * OUT_ROW * 4;

// WP by WQ waves of PB by QB blocks each, KW times: with KW = 2 each half of a k-tile is another wave's, and the two's sums meet in
// LDS at the end. STAGES k-tiles in LDS.
template <class T, bool PTR, bool QTR, int WP, int WQ, int PB, int QB, int KW, int STAGES>
struct Gemm {
    static constexpr int TP = 16 * PB * WP, TQ = 16 * QB * WQ, WAVES = WP * WQ * KW, THREADS = 64 * WAVES;
    typedef Side<PTR, TP, WAVES> P;
    typedef Side<QTR, TQ, WAVES> Q;
    static constexpr int STAGE = P::BYTES + Q::BYTES, JOIN = KW == 1 ? 0 : WP * WQ * PB * QB * 1024;
    static constexpr int STAGES_BYTES = STAGES * STAGE;
    static constexpr int OUT = WP * WQ * OUT_BYTES;
    static constexpr int LDS = STAGES_BYTES > JOIN ? STAGES_BYTES > OUT ? STAGES_BYTES : OUT : JOIN > OUT ? JOIN : OUT;

    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
    static __device__ __forceinline__ int wp() { return wave() % WP; }
    static __device__ __forceinline__ int wq() { return wave() / WP % WQ; }
    static __device__ __forceinline__ int kw() { return wave() / (WP * WQ); }

    // Lane c + 16 g: acc[b][q][i] belongs to p = 16 b + 4 g + i of the wave's 16 PB and row 16 q + c of its 16 QB.
    // With KW = 2 the sums are those of the waves with kw() = 0; the others return false.
    //
    // The barrier of a k-tile lies where a wave has read all it needs of it: its place then takes the k-tile STAGES further, and the
    // next one's first operands are read while the last products of this one run.
    //
    // begin() asks for the first k-tiles, run() does the rest. under: each wave has made UNDER other requests between the two, which
    // need not be waited for (requests end in their order).
    static __device__ __forceinline__ void begin(const P& p, const Q& q, char* lds, int kt0, int kt1)
    {
#pragma unroll
        for (int i = 0; i < STAGES; ++i)
            if (kt0 + i < kt1) {
                p.template bring<false>(lds + i * STAGE, kt0 + i);
                q.template bring<false>(lds + i * STAGE + P::BYTES, kt0 + i);
            }
    }
    template <int UNDER = 0>
    static __device__ __forceinline__ bool run(f32x4 (&acc)[PB][QB], const P& p, const Q& q, char* lds, int kt0, int kt1, bool under = false)
    {
#ifdef __HIP_DEVICE_COMPILE__
        const int half = KW == 2 ? kw() : 0;
        Reader<PTR, TP, PB> rp;
        Reader<QTR, TQ, QB> rq;
        rp.init(PB * wp(), half);
        rq.init(QB * wq(), half);
        u16x8 a[2][PB], b[2][QB];
        auto read = [&](int set, const char* from, int step) {
#pragma unroll
            for (int i = 0; i < PB; ++i) a[set][i] = rp.read(from, step, i);
#pragma unroll
            for (int i = 0; i < QB; ++i) b[set][i] = rq.read(from + P::BYTES, step, i);
        };
        auto products = [&](int set) {
#pragma unroll
            for (int j = 0; j < QB; ++j)
#pragma unroll
                for (int i = 0; i < PB; ++i) acc[i][j] = T::mfma(a[set][i], b[set][j], acc[i][j]);
        };
        auto bring = [&](int slot, int kt, auto whole) {
            p.template bring<decltype(whole)::value>(lds + slot, kt);
            q.template bring<decltype(whole)::value>(lds + slot + P::BYTES, kt);
        };
        constexpr int LOADS = P::LOADS + Q::LOADS;
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        // The order within a phase: the next products' operands are read between these.
        auto mix = [&] {
            constexpr int READS = (PTR ? 2 : 1) * PB + (QTR ? 2 : 1) * QB, EACH = PB * QB / READS > 1 ? 2 : 1;
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, PB * QB - EACH * READS, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        // k-tile kt has come for all waves, of which later ones are under way
        bool early = under;                             // nothing has been asked for since
        auto come = [&](auto later) {
            constexpr int OPEN = decltype(later)::value * LOADS;
            if (UNDER && early) wait_loads<OPEN + UNDER>();
            else wait_loads<OPEN>();
            arrive();
        };
        if (kt0 < kt1) {
            if (kt0 + STAGES - 1 < kt1) come(std::integral_constant<int, STAGES - 1>());
            else come(std::integral_constant<int, 0>());
            int now = 0, kt = kt0;
            // the k-tile that takes this one's place (more: it is whole), the next one's first operands, and the products of a set
            auto turn_over = [&](int set, auto more) {
                constexpr bool MORE = decltype(more)::value;
                come(std::integral_constant<int, MORE ? STAGES - 2 : 0>());
                early = early && kt + STAGES >= kt1;
                const int free = now;
                now = now == (STAGES - 1) * STAGE ? 0 : now + STAGE;
                // at once: spread over the products they come too late (8192 x 7168 x 4096: 406 us against 365)
                if constexpr (MORE) bring(free, kt + STAGES, yes);
                else if (kt + STAGES < kt1) bring(free, kt + STAGES, no);
                __builtin_amdgcn_sched_barrier(0);
                read(set ^ 1, lds + now, 0);                // behind the last k-tile: what is there, for no product
                products(set);
                mix();
                ++kt;
            };
            const int whole = (p.whole() < q.whole() ? p.whole() : q.whole()) < kt1 ? (p.whole() < q.whole() ? p.whole() : q.whole()) : kt1;
            if constexpr (KW == 1) {
                auto step = [&](auto more) {
                    read(1, lds + now, 1);
                    products(0);
                    mix();
                    turn_over(1, more);
                };
                read(0, lds, 0);
                while (kt + STAGES < whole) step(yes);
                while (kt < kt1) step(no);
            } else {
                read(0, lds, 0);
                while (kt + 1 + STAGES < whole) {
                    turn_over(0, yes);
                    turn_over(1, yes);
                }
                while (kt + 1 < kt1) {
                    turn_over(0, no);
                    turn_over(1, no);
                }
                if (kt < kt1) turn_over(0, no);
            }
        }
        __syncthreads();
        if constexpr (KW == 2) {
            f32x4* join = (f32x4*)lds + (wave() % (WP * WQ)) * (PB * QB * 64) + (threadIdx.x & 63);
            if (half) {
#pragma unroll
                for (int i = 0; i < PB; ++i)
#pragma unroll
                    for (int j = 0; j < QB; ++j) join[(i * QB + j) * 64] = acc[i][j];
            }
            __syncthreads();
            if (!half) {
#pragma unroll
                for (int i = 0; i < PB; ++i)
#pragma unroll
                    for (int j = 0; j < QB; ++j) acc[i][j] += join[(i * QB + j) * 64];
            }
            __syncthreads();
            return !half;
        }
#endif
        return true;
    }
};

// Two blocks of 16 values of a row, four a lane, to eight in a row a lane: lanes 16 apart exchange halves. Lane c + 16 g gets values
// 16 (g & 1) + 8 (g >> 1) .. + 7 of the 32.
template <class T>
__device__ __forceinline__ u16x8 paired(f32x4 a, f32x4 b)
{
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 o = {};
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t x = T::put(a[2 * i]) | (uint32_t)T::put(a[2 * i + 1]) << 16, y = T::put(b[2 * i]) | (uint32_t)T::put(b[2 * i + 1]) << 16;
        const auto s = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        o[i] = s[0];
        o[2 + i] = s[1];
    }
#endif
    return __builtin_bit_cast(u16x8, o);
}

// Four blocks of 16 values of a row to stores of whole lines: lanes 8 apart exchange what belongs to the first and the last 8 of the 16
// rows. Lane c + 16 g gets values 32 (c / 8) + 16 (g & 1) + 8 (g / 2) .. + 7 of the 64, of row c % 8 (v[0]) and 8 + c % 8 (v[1]). Stores of
// 64 bytes a row reach 3.7 TB/s, of 128 bytes 5.4.
template <class T>
__device__ __forceinline__ void lined(const f32x4 (&a)[4], u16x8 (&v)[2])
{
#ifdef __HIP_DEVICE_COMPILE__
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 x = __builtin_bit_cast(u32x4, paired<T>(a[0], a[1])), y = __builtin_bit_cast(u32x4, paired<T>(a[2], a[3]));
    const bool first = (threadIdx.x & 8) == 0;
    u32x4 p, q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t got = __builtin_amdgcn_update_dpp(0, first ? y[i] : x[i], 0x128, 0xf, 0xf, true);    // row_ror:8
        p[i] = first ? x[i] : got;
        q[i] = first ? got : y[i];
    }
    v[0] = __builtin_bit_cast(u16x8, p);
    v[1] = __builtin_bit_cast(u16x8, q);
#endif
}

// A wave's results by way of LDS: 16 PB columns of 64 rows at a time, rows OUT_ROW floats apart, so that neighbours get neighbouring
// values of a row (whole lines are loaded and stored) and the code that takes them is there once. f(rows in LDS, the first one's
// number in the wave's 16 QB, how many).
template <int PB, int QB, class F>
__device__ __forceinline__ void rows_of(const f32x4 (&acc)[PB][QB], char* lds, int slot, F f)
{
    static_assert(PB == 4);
    constexpr int QH = QB < 4 ? QB : 4;
    float* mine = (float*)(lds + slot * OUT_BYTES);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < QB / QH; ++half) {
#pragma unroll
        for (int j = 0; j < QH; ++j)
#pragma unroll
            for (int i = 0; i < PB; ++i) *(f32x4*)(mine + (16 * j + c) * OUT_ROW + 16 * i + 4 * g) = acc[i][half * QH + j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        f(mine, half * QH * 16, QH * 16);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

}  // namespace evamx_dense
