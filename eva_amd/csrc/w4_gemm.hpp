// The larger products on 4-bit weights: 64 rows by 256 columns a workgroup on v_mfma_f32_16x16x32_f16.
//
// Each of the four waves owns 64 columns (four streams of 16) for all 64 rows, so a weight is decoded once per 64 rows and by
// one wave only: codes go from memory to registers, two k-tiles ahead, and from there to the matrix cores (w4.hpp's layout). The
// rows' k-tile (16 KiB, of two halves 32) comes to LDS directly, into w4g_stages places in turn; its 16-byte chunks are swapped by
// the row's low bits (chunk c of row r lies at c ^ (r & 15)), so that the 16 rows of an operand are read from 16 different banks'
// quads. The direct load writes its lanes' pieces one after the other, so the swap is made in the addresses it reads.
//
// Per k-tile and wave: 64 matrix instructions (1024 cycles; 128 for rows of two halves), 144 to decode, 64 to add the groups' sums
// times their scales (256 with groups of 32), 16 reads of 1 KiB from LDS (32).
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

// Stages of the rows' LDS, of one half a value or of two (HL): with two, two stages of 32 KiB, so that two workgroups share a CU
// as with three of 16 (a layer of 1250 tokens, 39 rows an expert: 1750 us; with three of 32, one workgroup a CU, 1990).
template <bool HL>
constexpr int w4g_stages() { return HL ? 2 : 3; }
template <bool HL>
constexpr int w4g_lds() { return w4g_stages<HL>() * W4G_STAGE * (HL ? 2 : 1); }

// acc[b][mb]: rows 16 mb + 4 g + i of the tile at column c of stream b (lane c + 16 g). lds: w4g_lds<HL>() bytes.
//
// A k-tile is four phases of 32 k, or with HL eight, the values' first halves and their second ones in turn, whose weights are
// decoded once. A phase's 16 matrix instructions run while the wave reads and decodes the next phase's operands, so that neither
// LDS nor the vector instructions are waited for; the k-tile's last phase crosses to the next k-tile: its barrier lies before that
// phase, when the wave has read all it needs of the old tile. Codes come two k-tiles ahead, rows as many as there are stages.
template <int SG, bool ZERO, bool HL, int MB, int NB>
__device__ __forceinline__ void w4g_run(w4_f32x4 (&acc)[NB][MB], const W4Stream (&st)[NB], const W4GemmRows<MB>& rows, char* lds, int kt_n,
                                        int bf16)
{
#ifdef __HIP_DEVICE_COMPILE__                                          // the host pass does not know the builtins' operands
    constexpr int HALVES = HL ? 2 : 1, SLOT = HALVES * W4G_STAGE, STAGES = w4g_stages<HL>(), PHASES = 4 * HALVES;
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
    w4_half8 x[2][MB], w[2][NB];                                       // of phases and of their 32 k, in turn
    w4_f32x4 part[NB][MB];
    const int row_off = (lane & 15) * (W4_TILE_K * 2);
    auto read = [&](int slot, int q) {                                 // phase q's rows
        const char* at = lds + slot + row_off + (((4 * (q / HALVES) + (lane >> 4)) ^ (lane & 15)) * 16) + q % HALVES * W4G_STAGE;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) x[q & 1][mb] = *(const w4_half8*)(at + mb * (16 * W4_TILE_K * 2));
    };
    auto decode = [&](int j, const W4Raw<SG> (&r)[NB], int b0, int b1) {   // the weights of streams b0 .. b1 - 1 at the 32 k of j
#pragma unroll
        for (int b = b0; b < b1; ++b)
            w[j & 1][b] = w4_operand(r[b].c[j], w4_zero(ZERO ? (r[b].z >> (8 * (j * SG / 4))) & W4_ZERO_MAX : 8), consts);
    };
    auto products = [&](int q, const W4Raw<SG> (&r)[NB]) {
        constexpr int PER = PHASES / SG;                               // phases of a group
        const bool first = q % PER == 0, last = q % PER == PER - 1;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
                part[b][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[q & 1][mb], w[q / HALVES & 1][b], first ? w4_f32x4{0, 0, 0, 0} : part[b][mb],
                                                                     0, 0, 0);
        if (last) {
            const int g = q / PER;
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
        constexpr int VALU = ZERO ? 1 : 8 / MB;
        __builtin_amdgcn_sched_group_barrier(0x100, MB, 0);            // LDS reads, then matrix and vector instructions in turn
#pragma unroll
        for (int i = 0; i < NB * MB; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrive = [&] {                                                // all waves are here, and their LDS reads are done
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
    w4g_wait<ROWS + CODES>();                                          // the first k-tile's rows and codes are there
    arrive();
    if constexpr (STAGES == 3) bring(2 * SLOT, 2);
    read(0, 0);
    decode(0, raw[0], 0, NB);
    int now = 0;
    auto step = [&](int kt, W4Raw<SG> (&r)[NB], W4Raw<SG> (&ahead)[NB]) {
        const int next = now == (STAGES - 1) * SLOT ? 0 : now + SLOT;
#pragma unroll
        for (int q = 0; q < PHASES - 1; ++q) {
            const int j = q / HALVES, h = q % HALVES;
            read(now, q + 1);
            if (j < 3) decode(j + 1, r, h * NB / HALVES, (h + 1) * NB / HALVES);
            products(q, r);
            mix();
        }
        // requests under way: with three stages the rows of kt + 1, the codes of kt + 1 and the rows of kt + 2, in this order,
        // with two the codes and rows of kt + 1; what kt + 1 needs has to be there
        w4g_wait<STAGES == 3 ? ROWS : 0>();
        arrive();
        read(next, 0);
        decode(0, ahead, 0, NB);
        products(PHASES - 1, r);
        mix();
#pragma unroll
        for (int b = 0; b < NB; ++b) w4_load<SG, ZERO>(r[b], st[b], kt + 2);
        bring(now, kt + STAGES);
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
