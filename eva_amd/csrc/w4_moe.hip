// The routed (and shared) SwiGLU experts of an MoE layer on 4-bit weights with group scales (w4.hpp):
//   out[t] = sum_k w_tk D_e h_tk,  h = min(silu(G_e x_t), L) * clamp(U_e x_t, -L, L),  e = sel[t][k] - first_expert,
// over the slots whose e lies in [0, n_local); the shared experts are the last matrices of the stacks, weight 1, every token,
// their gate clamped before SiLU (both as evamx_moe_forward has them). L = 0: no clamping.
#include <cmath>

#include "evamx_gemv.hpp"
#include "evamx_internal.hpp"
#include "w4_gemm.hpp"

namespace evamx {

struct W4Unit {
    int expert, r0, rows, pad;   // rows slots from order[r0] on, all of one expert; expert -1: none
};

struct W4MoeParams {
    int rows, topk, n_shared, kt_slots, slots, n_local, count, hidden, inter, bf16;   // kt_slots = topk + n_shared per token
    uint32_t recip;              // ceil(2^32 / kt_slots)
    long long first;
    float limit;
    const int64_t* sel;
    const float* weights;
    W4Unit *units, *big;         // of up to 16 rows (W4_UNIT_ROWS) and up to 64 (W4G_ROWS)
    const int* units_in_use;     // number of the former, or NULL: one for each slot
    int* n_units;                // [2]
    int* order;                  // slots by (expert, slot)
    const void* x_in;            // as given
    size_t x_stride;
    int aligned;
    const w4_half* x;            // [rows][k of gate, padded], with a factor per row (NULL: 1)
    const float* xs;
    float* h;                    // [slots][h_ld]
    int h_ld;
    w4_half* hh;                 // the same, ready for the down products, with a factor per row
    float* hs;
    float* y;                    // [slots][hidden]
    void* out;
    size_t out_stride;
};

// Token of a slot: a division by a constant of the call as one high product (exact below 2^16).
__device__ __forceinline__ int w4_token(const W4MoeParams& p, int s) { return p.kt_slots == 1 ? s : (int)__umulhi((uint32_t)s, p.recip); }

// Matrix of slot s, or -1.
__device__ __forceinline__ int w4_slot_expert(const W4MoeParams& p, int s)
{
    int at = s;
    if (p.n_shared) {
        const int t = w4_token(p, s), k = s - t * p.kt_slots;
        if (k >= p.topk) return p.n_local + k - p.topk;
        at = t * p.topk + k;
    }
    const unsigned long long e = (unsigned long long)p.sel[at] - (unsigned long long)p.first;    // wraps
    return e < (unsigned)p.n_local ? (int)e : -1;
}

// What a call of more than W4_FEW_ROWS tokens needs before its products, one launch: workgroups 0 .. count - 1 group the slots
// stably by expert and cut each expert's into units; the others make a row of x ready each. An expert of at most `small` rows has
// units of 16 rows, one of more units of 64 (the last of any size). In a call of up to 16 tokens all are of 16, whatever an expert
// gets: a token's arithmetic is then the one it has alone.
//
// The workgroup of expert e reads every slot (from L2; far below the products that follow): a histogram gives the places of its
// slots and units, each wave counts its own range's slots of e, then writes them in order.
constexpr int W4_PREP_THREADS = 512, W4_UNIT_ROWS = 16;

// Experts of up to this many rows go to the kernels of 16-row units, which keep more of the memory busy; larger ones would read
// their weights twice there (7168 x 2048, 256 experts of 19 rows on average: 1365 us with 16, 1684 with 24; of 9 rows: 1298 and
// 1248).
constexpr int W4_REST_ROWS = 16;

template <int SRC>
__global__ __launch_bounds__(W4_PREP_THREADS) void w4_prep_kernel(W4MoeParams p, int small, w4_half* __restrict__ xh, float* __restrict__ xs, int n_pad)
{
    constexpr int WAVES = W4_PREP_THREADS / 64;
    __shared__ uint32_t top[WAVES];
    if ((int)blockIdx.x >= p.count) {
        const int t = blockIdx.x - p.count;
        W4ReadyRow<SRC, W4_PREP_THREADS, false> row{(const char*)p.x_in + t * p.x_stride * 2, p.hidden, n_pad, (bool)p.aligned, (int)threadIdx.x};
        row.load();
        const float f = row.finish(xh + (size_t)t * n_pad, 0, top);
        if (threadIdx.x == 0) xs[t] = f;
        return;
    }
    __shared__ int hist[1024], mine_n[WAVES], sums[5][WAVES];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < p.count; i += W4_PREP_THREADS) hist[i] = 0;
    __syncthreads();
    const int span = (w4_ceil(p.slots, WAVES) + 63) & ~63, s0 = wave * span, s1 = s0 + span < p.slots ? s0 + span : p.slots;
    int own = 0;
    for (int s = s0 + lane; s < s1; s += 64) {
        const int x = w4_slot_expert(p, s);
        if (x >= 0) atomicAdd(&hist[x], 1);
        own += x == e;
    }
    for (int i = 32; i; i >>= 1) own += __shfl_xor(own, i);
    if (lane == 0) mine_n[wave] = own;
    __syncthreads();
    auto bigs = [&](int n) { return n <= small ? 0 : (n + W4G_ROWS - 1) / W4G_ROWS; };
    auto smalls = [&](int n) { return n <= small ? (n + W4_UNIT_ROWS - 1) / W4_UNIT_ROWS : 0; };
    int v[5] = {0, 0, 0, 0, 0};                              // before e: slots, units, big units; in all: units, big units
    for (int i = threadIdx.x; i < p.count; i += W4_PREP_THREADS) {
        const int n = hist[i], u = smalls(n), b = bigs(n);
        v[3] += u;
        v[4] += b;
        if (i < e) {
            v[0] += n;
            v[1] += u;
            v[2] += b;
        }
    }
#pragma unroll
    for (int c = 0; c < 5; ++c) {
        for (int i = 32; i; i >>= 1) v[c] += __shfl_xor(v[c], i);
        if (lane == 0) sums[c][wave] = v[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 5; ++c) {
        v[c] = 0;
        for (int w = 0; w < WAVES; ++w) v[c] += sums[c][w];
    }
    const int n = hist[e], slots = v[0], nb = bigs(n), done = nb ? n : 0;
    if (e == 0 && threadIdx.x == 0) {
        p.n_units[0] = v[3];
        p.n_units[1] = v[4];
    }
    for (int i = threadIdx.x; i < nb; i += W4_PREP_THREADS)
        p.big[v[2] + i] = W4Unit{e, slots + i * W4G_ROWS, n - i * W4G_ROWS < W4G_ROWS ? n - i * W4G_ROWS : W4G_ROWS, 0};
    for (int i = threadIdx.x; done + i * W4_UNIT_ROWS < n; i += W4_PREP_THREADS) {
        const int r = done + i * W4_UNIT_ROWS;
        p.units[v[1] + i] = W4Unit{e, slots + r, n - r < W4_UNIT_ROWS ? n - r : W4_UNIT_ROWS, 0};
    }
    int at = slots;
    for (int w = 0; w < wave; ++w) at += mine_n[w];
    for (int b0 = s0; b0 < s1; b0 += 64) {
        const int s = b0 + lane;
        const bool mine = s < s1 && w4_slot_expert(p, s) == e;
        const unsigned long long b = __ballot(mine);
        if (mine) p.order[at + __popcll(b & ((1ull << lane) - 1))] = s;
        at += __popcll(b);
    }
}

__device__ __forceinline__ float w4_clamp(float v, float lo, float hi) { return v < lo ? lo : v > hi ? hi : v; }    // NaN stays

__device__ __forceinline__ float w4_swiglu(float g, float u, float limit, bool shared)
{
    if (limit != 0.0f) {
        u = w4_clamp(u, -limit, limit);
        if (shared && g > limit) g = limit;
    }
    float a = g / (1.0f + __expf(-g));
    if (limit != 0.0f && !shared && a > limit) a = limit;
    return a * u;
}

// Waves of a workgroup: parts of the k-tiles times column groups. The parts depend on the matrix alone (w4_part_begin), and a
// wave has at least some twenty tiles to make up for its start.
constexpr int W4_WAVES = 4;
inline int w4_moe_parts(int kt) { return kt >= 48 ? 4 : kt >= 24 ? 2 : 1; }

// Column tiles a wave takes at once, of gate and up each and of down. The rows' operands come from L2 with every tile, four
// times the bytes of one column tile's codes, so more columns for the same operands win (16 tokens of a 7168 x 2048 layer of
// 256 experts: 405 us with 1 and 2, 391 with 1 and 4, 369 with 2 and 4), while tiles requested further ahead cost the
// registers of waves that hide more (with two tiles in flight a stream instead of one: 374 us, with four 442).
constexpr int W4_GU_CT = 2, W4_DOWN_NB = 4;

// Up to W4_FEW_ROWS tokens whose rows a workgroup can stage (w4_stage_fits: 2 tokens of 7168 features), without a launch before it:
// 16 columns of gate and up of one expert a column group, the rows in LDS (w4_linear_few_kernel's scheme). Unit u is the expert of
// slot u, if no slot before it has that expert; with one token every slot is a unit. One token of a 7168 x 2048 layer with eight
// experts and a shared one: 28.6 us for 136 MB, 4.8 TB/s; reading as much with no decode takes 26.
constexpr int W4_FEW_ROWS = 4, W4_FEW_SLOTS = W4_FEW_ROWS * 64;

template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4_WAVES) void w4_gate_up_few_kernel(W4MoeParams p, W4Mat gate, W4Mat up, int parts)
{
    extern __shared__ w4_half xs[];
    __shared__ uint32_t top[W4_MAX_PARTS][4];
    __shared__ float scale[4], part[W4_WAVES][2][64];
    __shared__ int list[W4_FEW_SLOTS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = W4_WAVES / parts, ld = gate.kt * W4_TILE_K + W4_STAGE_PAD;
    const int q = wave % parts, nt = blockIdx.x * groups + wave / parts;
    const int k0 = w4_part_begin(gate.kt, parts, q), k1 = w4_part_begin(gate.kt, parts, q + 1);
    const int e = __builtin_amdgcn_readfirstlane(w4_slot_expert(p, blockIdx.y));
    W4Stage stage{(const uint16_t*)p.x_in, p.x_stride, p.rows, gate.n_in, gate.kt, p.bf16, p.aligned};
    stage.load();
    const bool tell = blockIdx.x == 0 && wave == 0;           // the down products take the units from here
    if (e < 0) {
        if (tell && lane == 0) p.units[blockIdx.y] = W4Unit{-1, 0, 0, 0};
        return;
    }
    int rows = 1;
    if (p.rows == 1) {
        list[0] = blockIdx.y;
    } else {
        rows = 0;
        bool first = true;
        int v[W4_FEW_ROWS];
#pragma unroll
        for (int c = 0; c < W4_FEW_ROWS; ++c) v[c] = 64 * c + lane < p.slots ? w4_slot_expert(p, 64 * c + lane) : -1;
#pragma unroll
        for (int c = 0; c < W4_FEW_ROWS; ++c) {
            const unsigned long long b = __ballot(v[c] == e);
            const int below = (int)blockIdx.y - 64 * c;
            if (v[c] == e) list[rows + __popcll(b & ((1ull << lane) - 1))] = 64 * c + lane;
            rows += __popcll(b);
            if (below >= 64 ? b != 0 : below > 0 && (b & ((1ull << below) - 1)) != 0) first = false;
        }
        if (!first) {
            if (tell && lane == 0) p.units[blockIdx.y] = W4Unit{-1, 0, 0, 0};
            return;
        }
    }
    wave_lds_fence();
    if (tell) {
        if (lane == 0) p.units[blockIdx.y] = W4Unit{e, (int)blockIdx.y * p.slots, rows, 0};
        for (int i = lane; i < rows; i += 64) p.order[blockIdx.y * p.slots + i] = list[i];
    }
    const int ntc = nt < gate.nt ? nt : gate.nt - 1;
    const W4Stream st[2] = {w4_stream<SG, ZERO>(gate, e, ntc, k1), w4_stream<SG, ZERO>(up, e, ntc, k1)};
    auto block = [&](int r0, auto begin) {
        const int mine = r0 + ((lane & 15) >> 2), token = w4_token(p, list[mine < rows ? mine : rows - 1]);
        const w4_half* a = xs + token * ld + 8 * (lane >> 4);
        w4_f32x4 acc[2][1] = {};
        w4_run<2, SG, ZERO, 2, 1, 1, false>(
            acc, st, k0, k1, gate.bf16, [](int, int) {},
            [&](int, int kt, w4_half8 (&x)[1][4], w4_half8 (&)[1][4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[0][j] = *(const w4_half8*)(a + kt * W4_TILE_K + 32 * j);
            },
            begin);
        part[wave][0][lane] = acc[0][0][0];
        part[wave][1][lane] = acc[1][0][0];
        __syncthreads();
        const int r = r0 + (lane >> 4), n = 16 * nt + (lane & 15);
        if (q == 0 && r < rows && n < p.inter) {
            float g = 0, v = 0;
            for (int w = 0; w < parts; ++w) {
                g += part[wave + w][0][lane];
                v += part[wave + w][1][lane];
            }
            const int s = list[r];
            const float f = scale[w4_token(p, s)];
            p.h[(size_t)s * p.h_ld + n] = w4_swiglu(g * f, v * f, p.limit, e >= p.n_local);
        }
        __syncthreads();
    };
    block(0, [&] { stage.finish(xs, top, scale); });
    for (int r0 = 4; r0 < rows; r0 += 4) block(r0, [] {});          // only where a token repeats an expert
}

// 16 W4_GU_CT columns of gate and up a column group, by a unit of up to 16 rows. 16 tokens of that layer, 82 experts: 237 us,
// 5.2 TB/s.
template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4_WAVES) void w4_gate_up_kernel(W4MoeParams p, W4Mat gate, W4Mat up, int parts)
{
    constexpr int CT = W4_GU_CT;
    __shared__ w4_f32x4 part[W4_WAVES][2 * CT][64];
    if ((int)blockIdx.y >= *p.units_in_use) return;
    const W4Unit u = p.units[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = W4_WAVES / parts;
    const int q = wave % parts, nt = CT * (blockIdx.x * groups + wave / parts);
    const int k0 = w4_part_begin(gate.kt, parts, q), k1 = w4_part_begin(gate.kt, parts, q + 1);
    W4Stream st[2 * CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int t = nt + c < gate.nt ? nt + c : gate.nt - 1;
        st[2 * c] = w4_stream<SG, ZERO>(gate, u.expert, t, k1);
        st[2 * c + 1] = w4_stream<SG, ZERO>(up, u.expert, t, k1);
    }
    W4GlobalRows<1, false> rows;
    rows.src = w4_rsrc(p.x, (uint32_t)p.rows * gate.kt * (W4_TILE_K * 2));
    const int mine = lane & 15, token = w4_token(p, p.order[u.r0 + (mine < u.rows ? mine : u.rows - 1)]);
    rows.at[0] = (uint32_t)token * gate.kt * (W4_TILE_K * 2) + 16 * (lane >> 4);
    w4_f32x4 acc[2 * CT][1] = {};
    w4_run<1, SG, ZERO, 2 * CT, 1, 4, false>(
        acc, st, k0, k1, gate.bf16, [&](int, int kt) { rows.request(kt); },
        [&](int, int, w4_half8 (&x)[1][4], w4_half8 (&lo)[1][4]) { rows.take(x, lo); }, [] {});
#pragma unroll
    for (int b = 0; b < 2 * CT; ++b) part[wave][b][lane] = acc[b][0];
    __syncthreads();
    for (int t = q; t < CT * 4; t += parts) {                // the parts share the values of their column group
        const int i = t & 3, c = t >> 2, r = 4 * (lane >> 4) + i, n = 16 * (nt + c) + (lane & 15);
        if (r >= u.rows || n >= p.inter) continue;
        float g = 0, v = 0;
        for (int w = wave - q; w < wave - q + parts; ++w) {
            g += part[w][2 * c][lane][i];
            v += part[w][2 * c + 1][lane][i];
        }
        const int s = p.order[u.r0 + r];
        const float f = p.xs ? p.xs[w4_token(p, s)] : 1.0f;
        p.h[(size_t)s * p.h_ld + n] = w4_swiglu(g * f, v * f, p.limit, u.expert >= p.n_local);
    }
}

// The hidden activations of the slots there are, ready for the down products, each as the sum of two halves: their first 11 bits,
// and what that rounding leaves, so that some 22 bits of them reach the results (relative error of an fp16 layer 2.9e-4 with one
// half, 2.1e-4 being the results' own rounding; bf16 results then differed by 9e-4 from those of fp32 arithmetic, now by 1e-5).
__global__ __launch_bounds__(256) void w4_hidden_kernel(W4MoeParams p, int n_pad)
{
    __shared__ uint32_t part[4];
    const int s = blockIdx.x;
    if (w4_slot_expert(p, s) < 0) return;
    W4ReadyRow<W4_SRC_F32, 256, true> row{(const char*)(p.h + (size_t)s * p.h_ld), p.inter, n_pad, true, (int)threadIdx.x};
    row.load();
    const float f = row.finish(p.hh + s * (size_t)(2 * n_pad), n_pad, part);
    if (threadIdx.x == 0) p.hs[s] = f;
}

// 16 W4_DOWN_NB columns of the output a column group, by a unit of up to 16 rows. 16 tokens as above: 146 us, 4.3 TB/s (127 with
// one half a value).
template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4_WAVES) void w4_down_kernel(W4MoeParams p, W4Mat down, int parts)
{
    constexpr int NB = W4_DOWN_NB;
    __shared__ w4_f32x4 part[W4_WAVES][NB][64];
    if (p.units_in_use && (int)blockIdx.y >= *p.units_in_use) return;
    const W4Unit u = p.units[blockIdx.y];
    if (u.expert < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = W4_WAVES / parts;
    const int q = wave % parts, nt = NB * (blockIdx.x * groups + wave / parts), n_pad = down.kt * W4_TILE_K;
    const int k0 = w4_part_begin(down.kt, parts, q), k1 = w4_part_begin(down.kt, parts, q + 1);
    W4Stream st[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c) st[c] = w4_stream<SG, ZERO>(down, u.expert, nt + c < down.nt ? nt + c : down.nt - 1, k1);
    W4GlobalRows<1, true> rows;
    const uint32_t ld = 4 * n_pad;
    rows.src = w4_rsrc(p.hh, (uint32_t)p.slots * ld);
    rows.lo_off = 2 * n_pad;
    for (int r0 = 0; r0 < u.rows; r0 += W4_UNIT_ROWS) {      // once, but for few tokens that repeat an expert
        const int mine = r0 + (lane & 15);
        rows.at[0] = (uint32_t)p.order[u.r0 + (mine < u.rows ? mine : u.rows - 1)] * ld + 16 * (lane >> 4);
        w4_f32x4 acc[NB][1] = {};
        w4_run<1, SG, ZERO, NB, 1, 4, true>(
            acc, st, k0, k1, down.bf16, [&](int, int kt) { rows.request(kt); },
            [&](int, int, w4_half8 (&x)[1][4], w4_half8 (&lo)[1][4]) { rows.take(x, lo); }, [] {});
#pragma unroll
        for (int c = 0; c < NB; ++c) part[wave][c][lane] = acc[c][0];
        __syncthreads();
        for (int t = q; t < NB * 4; t += parts) {
            const int i = t & 3, b = t >> 2, r = r0 + 4 * (lane >> 4) + i, n = 16 * (nt + b) + (lane & 15);
            if (r >= u.rows || n >= p.hidden) continue;
            float v = 0;
            for (int w = wave - q; w < wave - q + parts; ++w) v += part[w][b][lane][i];
            const int s = p.order[u.r0 + r];
            p.y[(size_t)s * p.hidden + n] = v * p.hs[s];
        }
        __syncthreads();
    }
}

// 128 columns of gate and up by a unit of up to 64 rows: the streams of a wave are gate and up of two column tiles. 2000 tokens of
// a 7168 x 2048 layer with groups of 32 and Zipf loads: 1409 us here and 382 in the small experts' kernel; with groups of 128 and
// even loads the whole layer runs at 650 TFLOP/s, of 8 slots a token. Three blocks of rows have a path of their own: 1250 tokens,
// 39 rows an expert, 1810 us against 1970 with four blocks; fp16 with groups of 64 and zero points 2100 against 2430.
template <int SG, bool ZERO, int MB>
__device__ __forceinline__ void w4_gate_up_gemm(const W4MoeParams& p, const W4Mat& gate, const W4Mat& up, const W4Unit& u, char* lds)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = (blockIdx.x * W4G_WAVES + wave) * (W4G_NB / 2);
    W4Stream st[W4G_NB];
#pragma unroll
    for (int c = 0; c < W4G_NB / 2; ++c) {
        const int t = nt + c < gate.nt ? nt + c : gate.nt - 1;
        st[2 * c] = w4_stream<SG, ZERO>(gate, u.expert, t, gate.kt);
        st[2 * c + 1] = w4_stream<SG, ZERO>(up, u.expert, t, gate.kt);
    }
    W4GemmRows<MB> rows;
    const uint32_t ld = gate.kt * (W4_TILE_K * 2);
    rows.src = w4_rsrc(p.x, p.rows * ld);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int r = w4g_row<MB>(i);
        rows.at[i] = w4_token(p, p.order[u.r0 + (r < u.rows ? r : u.rows - 1)]) * ld + w4g_chunk<MB>(i);
    }
    w4_f32x4 acc[W4G_NB][MB] = {};
    w4g_run<SG, ZERO, false, MB>(acc, st, rows, lds, gate.kt, gate.bf16);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 16 * mb + 4 * (lane >> 4) + i;
            if (r >= u.rows) continue;
            const int s = p.order[u.r0 + r];
            const float f = p.xs ? p.xs[w4_token(p, s)] : 1.0f;
#pragma unroll
            for (int c = 0; c < W4G_NB / 2; ++c) {
                const int n = 16 * (nt + c) + (lane & 15);
                if (n < p.inter)
                    p.h[(size_t)s * p.h_ld + n] = w4_swiglu(acc[2 * c][mb][i] * f, acc[2 * c + 1][mb][i] * f, p.limit, u.expert >= p.n_local);
            }
        }
}

template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4G_WAVES, 2) void w4_gate_up_gemm_kernel(W4MoeParams p, W4Mat gate, W4Mat up)
{
    __shared__ __attribute__((aligned(128))) char lds[w4g_lds<false>()];
    if ((int)blockIdx.y >= p.n_units[1]) return;
    const W4Unit u = p.big[blockIdx.y];
    if (u.rows > 48) w4_gate_up_gemm<SG, ZERO, 4>(p, gate, up, u, lds);
    else if (u.rows > 32) w4_gate_up_gemm<SG, ZERO, 3>(p, gate, up, u, lds);
    else if (u.rows > 16) w4_gate_up_gemm<SG, ZERO, 2>(p, gate, up, u, lds);
    else w4_gate_up_gemm<SG, ZERO, 1>(p, gate, up, u, lds);
}

// 256 columns of the output by a unit of up to 64 rows.
template <int SG, bool ZERO, int MB>
__device__ __forceinline__ void w4_down_gemm(const W4MoeParams& p, const W4Mat& down, const W4Unit& u, char* lds)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = (blockIdx.x * W4G_WAVES + wave) * W4G_NB;
    W4Stream st[W4G_NB];
#pragma unroll
    for (int b = 0; b < W4G_NB; ++b) st[b] = w4_stream<SG, ZERO>(down, u.expert, nt + b < down.nt ? nt + b : down.nt - 1, down.kt);
    W4GemmRows<MB> rows;
    const uint32_t half = down.kt * (W4_TILE_K * 2), ld = 2 * half;
    rows.src = w4_rsrc(p.hh, p.slots * ld);
    rows.lo_off = half;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int r = w4g_row<MB>(i);
        rows.at[i] = p.order[u.r0 + (r < u.rows ? r : u.rows - 1)] * ld + w4g_chunk<MB>(i);
    }
    w4_f32x4 acc[W4G_NB][MB] = {};
    w4g_run<SG, ZERO, true, MB>(acc, st, rows, lds, down.kt, down.bf16);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 16 * mb + 4 * (lane >> 4) + i;
            if (r >= u.rows) continue;
            const int s = p.order[u.r0 + r];
            const float f = p.hs[s];
#pragma unroll
            for (int b = 0; b < W4G_NB; ++b) {
                const int n = 16 * (nt + b) + (lane & 15);
                if (n < p.hidden) p.y[(size_t)s * p.hidden + n] = acc[b][mb][i] * f;
            }
        }
}

template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4G_WAVES, 2) void w4_down_gemm_kernel(W4MoeParams p, W4Mat down)
{
    __shared__ __attribute__((aligned(128))) char lds[w4g_lds<true>()];
    if ((int)blockIdx.y >= p.n_units[1]) return;
    const W4Unit u = p.big[blockIdx.y];
    if (u.rows > 48) w4_down_gemm<SG, ZERO, 4>(p, down, u, lds);
    else if (u.rows > 32) w4_down_gemm<SG, ZERO, 3>(p, down, u, lds);
    else if (u.rows > 16) w4_down_gemm<SG, ZERO, 2>(p, down, u, lds);
    else w4_down_gemm<SG, ZERO, 1>(p, down, u, lds);
}

// One token: 16 NB columns of the output, a wave a slot (up to 16, then the next ones), its parts of the k-tiles one after the
// other; the slots' sums meet in LDS, so that no launch follows. The layer above: 25.0 us for 68 MB, 2.7 TB/s; a wave's 32 KiB of
// codes are too few to make up for its start, and every value is read from LDS as two halves (20.3 with one; then 24.6 with 16
// columns a wave). Calls whose slots' activations do not fit W4_ONE_LDS take the general path: at nine slots of fp16 with groups of
// 64 and zero points 74.1 us, here 60.2; two slots of bf16 and 14336 105 here, of 16384 91 there.
constexpr int W4_ONE_WAVES = 16, W4_ONE_NB = 2, W4_ONE_LDS = 128 * 1024;

template <int SG, bool ZERO>
__global__ __launch_bounds__(64 * W4_ONE_WAVES) void w4_down_one_kernel(W4MoeParams p, W4Mat down, int parts)
{
    extern __shared__ w4_half hs[];                          // per wave, its slot's activations; then y[kt_slots][W4_ONE_NB][16]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, n_pad = down.kt * W4_TILE_K;
    w4_half* mine = hs + wave * (2 * n_pad);
    float (*y)[W4_ONE_NB][16] = (float (*)[W4_ONE_NB][16])(hs + waves * (2 * n_pad));
    const w4_half* a = mine + 8 * (lane >> 4);
    for (int s = wave; s < p.kt_slots; s += waves) {
        const int e = __builtin_amdgcn_readfirstlane(w4_slot_expert(p, s));
        if (e < 0) continue;
        W4ReadyRow<W4_SRC_F32, 64, true> row{(const char*)(p.h + (size_t)s * p.h_ld), p.inter, n_pad, true, lane};
        row.load();
        W4Stream st[W4_ONE_NB];
#pragma unroll
        for (int b = 0; b < W4_ONE_NB; ++b) {
            const int nt = W4_ONE_NB * blockIdx.x + b;
            st[b] = w4_stream<SG, ZERO>(down, e, nt < down.nt ? nt : down.nt - 1, down.kt);
        }
        float f = 0, v[W4_ONE_NB] = {};
        auto part = [&](int q, auto begin) {
            w4_f32x4 acc[W4_ONE_NB][1] = {};
            w4_run<2, SG, ZERO, W4_ONE_NB, 1, 1, true>(
                acc, st, w4_part_begin(down.kt, parts, q), w4_part_begin(down.kt, parts, q + 1), down.bf16, [](int, int) {},
                [&](int, int kt, w4_half8 (&x)[1][4], w4_half8 (&lo)[1][4]) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[0][j] = *(const w4_half8*)(a + kt * W4_TILE_K + 32 * j);
                        lo[0][j] = *(const w4_half8*)(a + n_pad + kt * W4_TILE_K + 32 * j);
                    }
                },
                begin);
#pragma unroll
            for (int b = 0; b < W4_ONE_NB; ++b) v[b] += acc[b][0][0];
        };
        part(0, [&] {
            f = row.finish(mine, n_pad, nullptr);
            wave_lds_fence();
        });
        for (int q = 1; q < parts; ++q) part(q, [] {});
        if (lane < 16)
#pragma unroll
            for (int b = 0; b < W4_ONE_NB; ++b) y[s][b][lane] = v[b] * f;
        wave_lds_fence();
    }
    __syncthreads();
    const int b = threadIdx.x >> 4, c = threadIdx.x & 15, n = 16 * (W4_ONE_NB * blockIdx.x + b) + c;
    if (threadIdx.x >= 16 * W4_ONE_NB || n >= p.hidden) return;
    float v = 0;
    for (int k = 0; k < p.kt_slots; ++k)
        if (w4_slot_expert(p, k) >= 0) v = __builtin_fmaf(k < p.topk ? p.weights[k] : 1.0f, y[k][b][c], v);
    w4_store(p.out, n, v, p.bf16);
}

// out[t] = the slots' outputs in slot order times their routing weights (fp32, as given), rounded once. Four columns a thread;
// the token's weights come first, so that all its slots' outputs are on their way at once.
__global__ __launch_bounds__(256) void w4_combine_kernel(W4MoeParams p)
{
    __shared__ float w[64];
    __shared__ int use[64];
    const int cols = (p.hidden + 1023) / 1024, t = blockIdx.x / cols, n = ((blockIdx.x - t * cols) * 256 + threadIdx.x) * 4;
    if ((int)threadIdx.x < p.kt_slots) {
        const int k = threadIdx.x;
        use[k] = w4_slot_expert(p, t * p.kt_slots + k) >= 0;
        w[k] = k < p.topk ? p.weights[(size_t)t * p.topk + k] : 1.0f;
    }
    __syncthreads();
    if (n >= p.hidden) return;
    const float* y = p.y + (size_t)t * p.kt_slots * p.hidden + n;
    float v[4] = {0, 0, 0, 0};
    if ((p.hidden & 3) == 0) {
#pragma unroll 8
        for (int k = 0; k < p.kt_slots; ++k) {
            if (!use[k]) continue;
            const w4_f32x4 a = *(const w4_f32x4*)(y + (size_t)k * p.hidden);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(w[k], a[i], v[i]);
        }
    } else {
        for (int k = 0; k < p.kt_slots; ++k)
            if (use[k])
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.hidden) v[i] = __builtin_fmaf(w[k], y[(size_t)k * p.hidden + i], v[i]);
    }
    for (int i = 0; i < 4; ++i)
        if (n + i < p.hidden) w4_store(p.out, (size_t)t * p.out_stride + n + i, v[i], p.bf16);
}

struct W4MoeLayout {
    size_t n_units, units, big, order, xs, x, h, hs, hh, y, total;
};

// The most units a call can have, whatever its routes: few tokens have one for each slot; else an expert has at most
// W4_REST_ROWS rows in units of 16, and one with units of 64 has more than W4_REST_ROWS rows for each.
static size_t w4_max_units(size_t slots, size_t count, bool few, bool all_small)
{
    if (few) return slots;
    const size_t rests = all_small ? (slots < count ? slots : count) + slots / W4_UNIT_ROWS : count * ((W4_REST_ROWS + W4_UNIT_ROWS - 1) / W4_UNIT_ROWS);
    return slots < rests ? slots : rests;
}

static size_t w4_max_big(size_t slots) { return slots / (W4_REST_ROWS + 1); }

static W4MoeLayout w4_moe_layout(int rows, int topk, int n_shared, int hidden, int inter)
{
    const size_t slots = (size_t)rows * (topk + n_shared);
    const size_t kx = (size_t)w4_ceil(hidden, W4_TILE_K) * W4_TILE_K, kh = (size_t)w4_ceil(inter, W4_TILE_K) * W4_TILE_K;
    W4MoeLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += w4_align(bytes); return o; };
    l.n_units = take(8);
    l.units = take(slots * sizeof(W4Unit));
    l.big = take(w4_max_big(slots) * sizeof(W4Unit));
    const size_t few = slots < W4_FEW_SLOTS ? slots : W4_FEW_SLOTS;   // units of few tokens have a list each; bytes grow with the rows
    l.order = take((few * few > slots ? few * few : slots) * 4);
    l.xs = take((size_t)rows * 4);
    l.x = take(rows * kx * 2);
    l.h = take(slots * kh * 4);
    l.hs = take(slots * 4);
    l.hh = take(slots * kh * 4);                             // two halves a value
    l.y = take(slots * hidden * 4);
    l.total = at;
    return l;
}

static bool w4_moe_shape_ok(int rows, int topk, int n_shared, int hidden, int inter, const char* who)
{
    if (topk < 1 || topk > 32 || n_shared < 0 || n_shared > 32) { set_error("%s: topk %d, n_shared %d outside 1..32, 0..32", who, topk, n_shared); return false; }
    if (rows < 1 || (long)rows * (topk + n_shared) > EVAMX_W4_MOE_MAX_SLOTS) {
        set_error("%s: %d rows of %d slots outside 1..%d slots", who, rows, topk + n_shared, EVAMX_W4_MOE_MAX_SLOTS);
        return false;
    }
    if (hidden < 1 || hidden > EVAMX_W4_MAX_DIM || inter < 1 || inter > EVAMX_W4_MAX_DIM) { set_error("%s: hidden %d or inter %d", who, hidden, inter); return false; }
    const long kx = w4_ceil(hidden, W4_TILE_K) * (long)W4_TILE_K, kh = w4_ceil(inter, W4_TILE_K) * (long)W4_TILE_K;
    if (rows * kx >= 1l << 31 || (long)rows * (topk + n_shared) * kh >= 1l << 30) {
        set_error("%s: %d rows of %d features or their hidden activations exceed 2^31 or 2^30 values", who, rows, hidden);
        return false;
    }
    return true;
}

}  // namespace evamx

using namespace evamx;

extern "C" size_t evamx_w4_moe_workspace_bytes(int rows, int topk, int n_shared, int hidden, int inter)
{
    return w4_moe_shape_ok(rows, topk, n_shared, hidden, inter, "evamx_w4_moe_workspace_bytes")
               ? w4_moe_layout(rows, topk, n_shared, hidden, inter).total : 0;
}

extern "C" int evamx_w4_moe_forward(const evamx_w4_moe_args* a, evamx_stream_t stream)
{
    static const char who[] = "evamx_w4_moe_forward";
    set_error("%s", "");
    if (!a) { set_error("%s: null arguments", who); return EVAMX_EINVAL; }
    if (!w4_weight_ok(a->gate, who) || !w4_weight_ok(a->up, who) || !w4_weight_ok(a->down, who)) return EVAMX_EINVAL;
    const evamx_w4_weight &g = *a->gate, &u = *a->up, &d = *a->down;
    if (g.count != u.count || g.count != d.count || g.n_in != u.n_in || g.n_out != u.n_out || d.n_in != g.n_out || d.n_out != g.n_in) {
        set_error("%s: gate %d x [%d, %d], up %d x [%d, %d] and down %d x [%d, %d] do not fit", who, g.count, g.n_out, g.n_in, u.count,
                  u.n_out, u.n_in, d.count, d.n_out, d.n_in);
        return EVAMX_EINVAL;
    }
    if (g.group != u.group || g.scale_dtype != u.scale_dtype || (g.zeros == nullptr) != (u.zeros == nullptr)) {
        set_error("%s: gate and up differ in their group size, scale type or zero points", who);
        return EVAMX_EINVAL;
    }
    if (!w4_moe_shape_ok(a->rows, a->topk, a->n_shared, g.n_in, g.n_out, who)) return EVAMX_EINVAL;
    if (a->n_shared > g.count) { set_error("%s: %d shared experts of %d", who, a->n_shared, g.count); return EVAMX_EINVAL; }
    if (!a->x || !a->sel || !a->weights || !a->out || !a->workspace) { set_error("%s: null pointer", who); return EVAMX_EINVAL; }
    if (a->x_dtype != EVAMX_DTYPE_F16 && a->x_dtype != EVAMX_DTYPE_BF16) { set_error("%s: x_dtype %d", who, a->x_dtype); return EVAMX_EINVAL; }
    if (a->x_stride < g.n_in || a->out_stride < g.n_in) { set_error("%s: strides below the row length", who); return EVAMX_EINVAL; }
    if (!(a->limit >= 0) || !std::isfinite(a->limit)) { set_error("%s: limit must be finite and >= 0", who); return EVAMX_EINVAL; }
    if ((uintptr_t)a->workspace & 15) { set_error("%s: the workspace must be 16-byte aligned", who); return EVAMX_EINVAL; }
    const W4MoeLayout l = w4_moe_layout(a->rows, a->topk, a->n_shared, g.n_in, g.n_out);
    if (a->workspace_bytes < l.total) { set_error("%s: workspace %zu bytes < %zu", who, a->workspace_bytes, l.total); return EVAMX_ENOSPACE; }

    char* ws = (char*)a->workspace;
    W4MoeParams p;
    p.rows = a->rows; p.topk = a->topk; p.n_shared = a->n_shared; p.kt_slots = a->topk + a->n_shared; p.slots = a->rows * p.kt_slots;
    p.count = g.count; p.n_local = g.count - a->n_shared; p.hidden = g.n_in; p.inter = g.n_out; p.bf16 = a->x_dtype == EVAMX_DTYPE_BF16;
    p.recip = (uint32_t)(((1ull << 32) + p.kt_slots - 1) / p.kt_slots);
    p.first = a->first_expert; p.limit = a->limit; p.sel = a->sel; p.weights = a->weights;
    p.n_units = (int*)(ws + l.n_units); p.units = (W4Unit*)(ws + l.units); p.big = (W4Unit*)(ws + l.big); p.order = (int*)(ws + l.order);
    p.x = (const w4_half*)(ws + l.x); p.xs = (const float*)(ws + l.xs);
    p.h = (float*)(ws + l.h); p.hh = (w4_half*)(ws + l.hh); p.hs = (float*)(ws + l.hs); p.y = (float*)(ws + l.y);
    p.out = a->out; p.out_stride = (size_t)a->out_stride;
    const hipStream_t s = (hipStream_t)stream;
    const W4Mat gm = w4_mat(g), um = w4_mat(u), dm = w4_mat(d);
    p.x_in = a->x; p.x_stride = (size_t)a->x_stride;
    p.aligned = (((uintptr_t)a->x | (uintptr_t)(2 * a->x_stride)) & 15) == 0;
    const int gp = w4_moe_parts(gm.kt), dp = w4_moe_parts(dm.kt), h_pad = dm.kt * W4_TILE_K;
    p.h_ld = h_pad;
    const bool few = w4_stage_fits(p.rows, gm.kt, W4_WAVES);
    const bool all_small = p.rows <= W4_UNIT_ROWS || p.slots <= W4_REST_ROWS;
    const unsigned units = (unsigned)w4_max_units(p.slots, p.count, few, all_small), bigs = few || all_small ? 0 : (unsigned)w4_max_big(p.slots);
    p.units_in_use = few ? nullptr : p.n_units;

    // a few tokens: their rows in LDS; one token: two launches in all
    if (few) {
        w4_dispatch(g, [&](auto sg, auto zero) {
            w4_gate_up_few_kernel<decltype(sg)::value, decltype(zero)::value>
                <<<dim3(w4_ceil(gm.nt, W4_WAVES / gp), units), 64 * W4_WAVES, w4_stage_bytes(p.rows, gm.kt), s>>>(p, gm, um, gp);
        });
        const int one_waves = p.kt_slots < W4_ONE_WAVES ? p.kt_slots : W4_ONE_WAVES;
        const size_t one_bytes = (size_t)one_waves * h_pad * 4 + (size_t)p.kt_slots * W4_ONE_NB * 16 * 4;
        if (p.rows == 1 && one_bytes <= W4_ONE_LDS) {
            w4_dispatch(d, [&](auto sg, auto zero) {
                w4_down_one_kernel<decltype(sg)::value, decltype(zero)::value>
                    <<<w4_ceil(dm.nt, W4_ONE_NB), 64 * one_waves, one_bytes, s>>>(p, dm, dp);
            });
            return launched("w4_moe_forward");
        }
    } else {
        const bool ready = w4_rows_ready(a->x, a->x_dtype, a->x_stride, p.hidden);
        const int blocks = p.count + (ready ? 0 : p.rows), x_pad = gm.kt * W4_TILE_K, rest = all_small ? p.slots : W4_REST_ROWS;
        w4_half* xh = (w4_half*)(ws + l.x);
        float* xs = (float*)(ws + l.xs);
        if (p.bf16) w4_prep_kernel<EVAMX_DTYPE_BF16><<<blocks, W4_PREP_THREADS, 0, s>>>(p, rest, xh, xs, x_pad);
        else w4_prep_kernel<EVAMX_DTYPE_F16><<<blocks, W4_PREP_THREADS, 0, s>>>(p, rest, xh, xs, x_pad);
        p.x = ready ? (const w4_half*)a->x : xh;
        p.xs = ready ? nullptr : xs;
        w4_dispatch(g, [&](auto sg, auto zero) {
            constexpr int SG = decltype(sg)::value;
            constexpr bool ZERO = decltype(zero)::value;
            if (bigs) w4_gate_up_gemm_kernel<SG, ZERO><<<dim3(w4_ceil(gm.nt, W4G_WAVES * W4G_NB / 2), bigs), 64 * W4G_WAVES, 0, s>>>(p, gm, um);
            w4_gate_up_kernel<SG, ZERO>
                <<<dim3(w4_ceil(gm.nt, W4_GU_CT * (W4_WAVES / gp)), units), 64 * W4_WAVES, 0, s>>>(p, gm, um, gp);
        });
    }
    w4_hidden_kernel<<<p.slots, 256, 0, s>>>(p, h_pad);
    w4_dispatch(d, [&](auto sg, auto zero) {
        constexpr int SG = decltype(sg)::value;
        constexpr bool ZERO = decltype(zero)::value;
        const dim3 grid(w4_ceil(dm.nt, W4_DOWN_NB * (W4_WAVES / dp)), units), big_grid(w4_ceil(dm.nt, W4G_WAVES * W4G_NB), bigs);
        if (bigs) w4_down_gemm_kernel<SG, ZERO><<<big_grid, 64 * W4G_WAVES, 0, s>>>(p, dm);
        w4_down_kernel<SG, ZERO><<<grid, 64 * W4_WAVES, 0, s>>>(p, dm, dp);
    });
    w4_combine_kernel<<<p.rows * w4_ceil(p.hidden, 1024), 256, 0, s>>>(p);
    return launched("w4_moe_forward");
}
