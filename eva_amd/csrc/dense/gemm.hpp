// The tiles of the larger products: acc[p][q] += sum_k P[p][k] Q[q][k] on v_mfma_f32_16x16x32.
//
// p runs along a row of the result (so that a lane ends up with eight values in a row), q over its rows. A matrix comes either
// with k along its rows in memory, or (TR) with k over its rows: then LDS holds it as it lies in memory and ds_read_b64_tr_b16
// turns it on the way to the registers. k-tiles of 64 come to LDS directly, two stages in turn.
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

// One matrix of a workgroup's product: N values of p or q, by k.
//   k along the rows:  value n is row map(n) of base, cut to `rows` rows, of `len` = K values.
//   TR:                k is the row, cut to `rows` = K rows; value n is column n of base, cut to `len` columns.
// In LDS in chunks of 16 bytes, in the order in which the direct loads write them; the chunks of a row are swapped by the row's low
// bits (in the addresses that are loaded), so that what an instruction reads together lies in different banks.
template <bool TR, int N, int WAVES, bool PERM, bool LOOSE>
struct Side {
    static constexpr int BYTES = N * TILE_K * 2, LOADS = BYTES / 1024 / WAVES, ROW_CHUNKS = TR ? N / 8 : TILE_K / 8;
    static_assert(LOADS >= 1 && LOADS * WAVES * 1024 == BYTES);
    const uint16_t* base;
    size_t stride;
    int rows, len;
    uint32_t at[LOADS];           // byte offsets of a lane's chunks (LOOSE: their row and first value, row << 8 | chunk)

    static __device__ __forceinline__ int swap(int row) { return TR ? (row & 3) << (PERM ? 2 : 1) : row & 7; }

    template <class Map>
    __device__ __forceinline__ void init(const uint16_t* b, size_t s, int r, int l, Map map)
    {
        base = b; stride = s; rows = r; len = l;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int slot = (i * WAVES + wave) * 64 + lane, row = slot / ROW_CHUNKS, chunk = (slot % ROW_CHUNKS) ^ swap(row);
            const int from = TR ? row : map(row);
            at[i] = LOOSE ? (uint32_t)from << 8 | chunk : (uint32_t)from * (uint32_t)stride * 2 + chunk * 16;
        }
    }
    // k-tile kt to LDS at `to`. Rows, columns and k that are not there become zeros; with TR, columns behind the last may hold the
    // next row's values, which end in results that are not stored.
    __device__ __forceinline__ void bring(char* to, int kt) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k0 = kt * TILE_K;
        if constexpr (LOOSE) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int row = (int)(at[i] >> 8) + (TR ? k0 : 0), v = (int)(at[i] & 255) * 8 + (TR ? 0 : k0);
                u16x8 x = (u16x8)(uint16_t)0;
                if (row < rows && v < len) {
                    const uint16_t* p = base + (size_t)row * stride + v;
                    if (v + 8 <= len) {
                        x = *(const u16x8_loose*)p;
                    } else {
#pragma unroll
                        for (int j = 0; j < 7; ++j)
                            if (v + j < len) x[j] = p[j];
                    }
                }
                *(u16x8*)(to + (i * WAVES + wave) * 1024 + lane * 16) = x;
            }
        } else if constexpr (TR) {
            const int left = rows - k0 < TILE_K ? rows - k0 : TILE_K;
            const __amdgpu_buffer_rsrc_t src = buffer(base + (size_t)k0 * stride, left <= 0 ? 0u : (uint32_t)((left - 1) * stride + len) * 2);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)(to + (i * WAVES + wave) * 1024), 16, at[i],
                                                         0, 0, 0);
        } else {
            const __amdgpu_buffer_rsrc_t src = buffer(base, rows <= 0 ? 0u : (uint32_t)((rows - 1) * stride + len) * 2);
            const int left = len - k0;                                  // chunks behind the row's end: no address
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int chunk = ((i * WAVES + wave) * 64 + lane) % ROW_CHUNKS ^ swap(((i * WAVES + wave) * 64 + lane) / ROW_CHUNKS);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)(to + (i * WAVES + wave) * 1024), 16,
                                                         chunk * 8 < left ? at[i] + (uint32_t)k0 * 2 : 0xfffffff0u, 0, 0, 0);
            }
        }
#endif
    }
};

// What a lane of a wave reads of a side: BLOCKS blocks of 16 values from block `first` on, lane c + 16 g the k 8 g .. 8 g + 7 of
// each 32. With PERM blocks come in pairs: value c of block b of a pair is p = 8 (c / 4) + 4 b + c % 4 of its 32 (k along the rows: the
// caller's map has put it there).
template <bool TR, int N, int BLOCKS, bool PERM>
struct Reader {
    static constexpr int BASES = !TR ? 2 : PERM ? BLOCKS / 2 : BLOCKS < 4 ? BLOCKS : 4;
    uint32_t at[BASES];

    __device__ __forceinline__ void init(int first)
    {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        if constexpr (!TR) {
            at[0] = (16 * first + c) * (TILE_K * 2) + ((g ^ (c & 7)) * 16);
            at[1] = at[0] ^ 64;
        } else {
            const int row = 8 * g + (c >> 2), low = row & 3;
#pragma unroll
            for (int j = 0; j < BASES; ++j) {
                const int chunk = PERM ? 4 * ((first / 2 + j) ^ low) + (c & 3) : 2 * ((first + j) ^ low) + ((c & 3) >> 1);
                at[j] = row * (N * 2) + chunk * 16 + (PERM ? 0 : 8 * (c & 1));
            }
        }
    }
    __device__ __forceinline__ u16x8 read(const char* lds, int step, int b) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        if constexpr (!TR) {
            return *(const u16x8*)(lds + at[step] + b * (16 * TILE_K * 2));
        } else {
            const char* p = lds + (PERM ? at[b >> 1] + 8 * (b & 1) : at[b & 3] + (b >> 2) * 128) + step * (32 * N * 2);
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * N * 2));
            return __builtin_bit_cast(u16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
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

// WP by WQ waves of PB by QB blocks each.
template <class T, bool PTR, bool QTR, int WP, int WQ, int PB, int QB, bool LOOSE>
struct Gemm {
    static constexpr int TP = 16 * PB * WP, TQ = 16 * QB * WQ, WAVES = WP * WQ;
    typedef Side<PTR, TP, WAVES, true, LOOSE> P;
    typedef Side<QTR, TQ, WAVES, false, LOOSE> Q;
    static constexpr int STAGE = P::BYTES + Q::BYTES, LDS = 2 * STAGE;

    // Lane c + 16 g: acc[2 j + b][q][i] belongs to p = 32 j + 8 g + 4 b + i of the wave's 16 PB and row 16 q + c of its 16 QB.
    // A k-tile is two phases of 32 k: while one's products run, the next one's operands are read; the barrier lies before the second,
    // when a wave has read all it needs of the k-tile, whose place the k-tile after the next then takes.
    static __device__ __forceinline__ void run(f32x4 (&acc)[PB][QB], const P& p, const Q& q, char* lds, int kt0, int kt1)
    {
#ifdef __HIP_DEVICE_COMPILE__
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        Reader<PTR, TP, PB, true> rp;
        Reader<QTR, TQ, QB, false> rq;
        rp.init(PB * (wave % WP));
        rq.init(QB * (wave / WP));
        u16x8 a[2][PB], b[2][QB];
        auto read = [&](int slot, int step) {
#pragma unroll
            for (int i = 0; i < PB; ++i) a[step][i] = rp.read(lds + slot, step, i);
#pragma unroll
            for (int i = 0; i < QB; ++i) b[step][i] = rq.read(lds + slot + P::BYTES, step, i);
        };
        auto products = [&](int step) {
#pragma unroll
            for (int j = 0; j < QB; ++j)
#pragma unroll
                for (int i = 0; i < PB; ++i) acc[i][j] = T::mfma(a[step][i], b[step][j], acc[i][j]);
        };
        auto bring = [&](int slot, int kt) {
            p.bring(lds + slot, kt);
            q.bring(lds + slot + P::BYTES, kt);
        };
        if (kt0 >= kt1) return;
        bring(0, kt0);
        if (kt0 + 1 < kt1) bring(STAGE, kt0 + 1);
        if (kt0 + 1 < kt1) wait_loads<LOOSE ? 0 : P::LOADS + Q::LOADS>();
        else wait_loads<0>();
        arrive();
        read(0, 0);
        int now = 0;
        for (int kt = kt0; kt < kt1; ++kt) {
            read(now, 1);
            products(0);
            wait_loads<0>();
            arrive();
            if (kt + 2 < kt1) bring(now, kt + 2);
            now ^= STAGE;
            if (kt + 1 < kt1) read(now, 0);
            products(1);
        }
#endif
    }
};

}  // namespace evamx_dense
