// The larger products on 4-bit weights: 64 rows by 256 columns a workgroup on v_mfma_f32_16x16x32_f16.
//
// Each of the four waves owns 64 columns (four streams of 16) for all 64 rows, so a weight is decoded once per 64 rows and by
// one wave only: codes go from memory to registers, a k-tile ahead, and from there to the matrix cores (w4.hpp's layout). The
// rows' k-tile (16 KiB) comes to LDS directly, double-buffered; its 16-byte chunks are swapped by the row's low bits (chunk c of
// row r lies at c ^ (r & 15)), so that the 16 rows of an operand are read from 16 different banks' quads. The direct load
// writes its lanes' pieces one after the other, so the swap is made in the addresses it reads.
//
// Per k-tile and wave: 64 matrix instructions (1024 cycles), 144 to decode, 64 to add the groups' sums times their scales (256
// with groups of 32), 16 reads of 1 KiB from LDS.
#pragma once
#include "w4.hpp"

namespace evamx {

// A tile of fewer rows is run as one of fewer blocks of 16 (MB): it brings, reads and multiplies no more.
constexpr int W4G_ROWS = 64, W4G_NB = 4, W4G_WAVES = 4;
constexpr int W4G_COLS = 16 * W4G_NB * W4G_WAVES;                   // 256
constexpr int W4G_STAGE = W4G_ROWS * W4_TILE_K * 2;                 // bytes of the rows' k-tile

// Columns of a lane: stream b of the wave, column c. Rows: 16 mb + 4 g + i (lane c + 16 g).
//
// Rows of a workgroup's tile of 16 MB: at[i] is the byte offset in src of the row that the lane brings with its i'th load (row
// w4g_row(i) of the tile), its 16-byte chunk included; for HL the same row's low half lies lo_off behind.
template <int MB>
struct W4GemmRows {
    __amdgpu_buffer_rsrc_t src;
    uint32_t at[MB], lo_off;
};

template <int MB>
__device__ __forceinline__ int w4g_row(int i) { return 4 * MB * (threadIdx.x >> 6) + 4 * i + ((threadIdx.x & 63) >> 4); }
template <int MB>
__device__ __forceinline__ uint32_t w4g_chunk(int i) { return (uint32_t)(((threadIdx.x & 15) ^ (w4g_row<MB>(i) & 15)) * 16); }

// s_waitcnt vmcnt(n) alone.
template <int N>
__device__ __forceinline__ void w4g_wait()
{
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | 15 << 8 | (N >> 4) << 14);
}

constexpr int W4G_STAGES = 3;

// acc[b][mb]: rows 16 mb + 4 g + i of the tile at column c of stream b (lane c + 16 g). lds: W4G_STAGES (HL: twice that) x
// W4G_STAGE bytes.
//
// A k-tile is four phases of 32 k. A phase's 16 matrix instructions run while the wave reads and decodes the next phase's
// operands, so that neither LDS nor the vector instructions are waited for; the k-tile's last phase crosses to the next k-tile:
// its barrier lies before that phase, when the wave has read all it needs of the old tile. Rows and codes come two to three
// k-tiles ahead.
template <int SG, bool ZERO, bool HL, int MB, int NB>
__device__ __forceinline__ void w4g_run(w4_f32x4 (&acc)[NB][MB], const W4Stream (&st)[NB], const W4GemmRows<MB>& rows, char* lds, int kt_n,
                                        int bf16)
{
#ifdef __HIP_DEVICE_COMPILE__                                          // the host pass does not know the builtins' operands
    constexpr int HALVES = HL ? 2 : 1, SLOT = HALVES * W4G_STAGE;
    constexpr int CODES = NB * (ZERO ? 3 : 2), ROWS = MB * HALVES;  // requests of a wave and k-tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const W4Consts consts;
    auto bring = [&](int slot, int kt) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int i = 0; i < MB; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rows.src,
                                                         (__attribute__((address_space(3))) void*)(lds + slot + h * W4G_STAGE + (wave * MB + i) * 1024),
                                                         16, rows.at[i] + (h ? rows.lo_off : 0u) + (uint32_t)kt * (W4_TILE_K * 2), 0, 0, 0);
    };
    W4Raw<SG> raw[2][NB];
    w4_half8 x[2][HALVES][MB], w[2][NB];
    w4_f32x4 part[NB][MB];
    const int row_off = (lane & 15) * (W4_TILE_K * 2);
    auto operands = [&](int to, int slot, int j, const W4Raw<SG> (&r)[NB]) {
        const char* at = lds + slot + row_off + (((4 * j + (lane >> 4)) ^ (lane & 15)) * 16);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) x[to][h][mb] = *(const w4_half8*)(at + h * W4G_STAGE + mb * (16 * W4_TILE_K * 2));
#pragma unroll
        for (int b = 0; b < NB; ++b) w[to][b] = w4_operand(r[b].c[j], w4_zero(ZERO ? (r[b].z >> (8 * (j * SG / 4))) & 15 : 8), consts);
    };
    auto products = [&](int from, int j, const W4Raw<SG> (&r)[NB]) {
        constexpr int PER = 4 / SG;                                    // phases of a group
        const bool first = j % PER == 0, last = j % PER == PER - 1;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                part[b][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[from][0][mb], w[from][b], first ? w4_f32x4{0, 0, 0, 0} : part[b][mb], 0, 0, 0);
                if constexpr (HL) part[b][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[from][HALVES - 1][mb], w[from][b], part[b][mb], 0, 0, 0);
            }
        }
        if (last) {
            const int g = j / PER;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float s = w4_scale((uint16_t)(r[b].s[g >> 1] >> (16 * (g & 1))), bf16);
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][mb][i] = __builtin_fmaf(part[b][mb][i], s, acc[b][mb][i]);
            }
        }
    };
    auto mix = [&] {                                                   // the order within a phase
        constexpr int READS = MB * HALVES, VALU = ZERO ? 1 : 8 / MB;
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);    // LDS reads, then matrix and vector instructions in turn
#pragma unroll
        for (int i = 0; i < 4 * MB * HALVES; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrive = [&] {                                                // all waves' rows of a k-tile are there, and its codes
        w4g_wait<ROWS + CODES>();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        bring(d * SLOT, d);
#pragma unroll
        for (int b = 0; b < NB; ++b) w4_load<SG, ZERO>(raw[d][b], st[b], d);
    }
    arrive();
    bring(2 * SLOT, 2);
    operands(0, 0, 0, raw[0]);
    int now = 0;
    auto step = [&](int kt, W4Raw<SG> (&r)[NB], W4Raw<SG> (&ahead)[NB]) {
        const int next = now == (W4G_STAGES - 1) * SLOT ? 0 : now + SLOT;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            operands((j + 1) & 1, now, j + 1, r);
            products(j & 1, j, r);
            mix();
        }
        // requests under way: the rows of kt + 1 and kt + 2, the codes of kt + 1 before those rows
        w4g_wait<ROWS>();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        operands(0, next, 0, ahead);
        products(1, 3, r);
        mix();
#pragma unroll
        for (int b = 0; b < NB; ++b) w4_load<SG, ZERO>(r[b], st[b], kt + 2);
        bring(now, kt + 3);
        now = next;
    };
    int kt = 0;
    for (; kt + 1 < kt_n; kt += 2) {
        step(kt, raw[0], raw[1]);
        step(kt + 1, raw[1], raw[0]);
    }
    if (kt < kt_n) step(kt, raw[0], raw[1]);
    w4g_wait<0>();                                                     // nothing may come into LDS after the workgroup's end
#endif
}

}  // namespace evamx
