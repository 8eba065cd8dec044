// Per-sequence expert counts and balance loss of a router, and the loss's gradient.
//
// Token t of sequence s has scores a_e = score(z_te) (the router's score function), shares p_e = a_e / sum a and topk picks
// sel. With n valid tokens and c_e picks of expert e in the sequence,
//   L_s = sum_e f_e P_e,  f_e = E c_e / (topk n),  P_e = (1/n) sum_t p_te       (1 where picks and shares are even).
// The counts are constants of the gradient:
//   dL_s/dz_tj = E / (topk n^2) * p_tj * (c_j - sum_i c_i p_ti) * dlog a_j/dz_j,
//   dlog a/dz = sigma(-z) for sigmoid, sigma(z) / (2 softplus(z)) for sqrt(softplus).
#include <cstring>

#include <type_traits>

#include "evamx_device.hpp"
#include "evamx_internal.hpp"

namespace evamx {

constexpr int BAL_MAX_EXPERTS = 512;

struct BalanceParams {
    const void* logits;
    int dtype, rows, experts, topk, sequences, score;
    size_t stride;
    const int64_t* sel;
    const int32_t* starts;      // [sequences + 1] or NULL: one sequence of all rows
    const uint8_t* mask;        // [rows] or NULL: nonzero where the token counts
    float* loss;                // [sequences]
    int32_t* counts;            // [sequences][experts]
    int32_t* tokens;            // [sequences]
    const float* grad_loss;
    void* grad;
    // work: chunks of `chunk` rows, a workgroup each; the part of sequence s in chunk w is piece w + s (an ascending walk over
    // both, so no two parts share one)
    int chunk;
    uint32_t recip;             // ceil(2^32 / topk)
    float* share;               // [pieces][experts]: sum of p
    int32_t* picks;             // [pieces][experts]
    int32_t* piece_tokens;      // [pieces]
    float* group_loss;          // [sequences][groups of 64 experts]
    unsigned long long* arrive; // [sequences], ARRIVE_STRIDE words apart
};

template <int DT>
__device__ __forceinline__ float bal_load(const void* p, size_t at)
{
    if constexpr (DT == EVAMX_DTYPE_F32) return ((const float*)p)[at];
    else if constexpr (DT == EVAMX_DTYPE_BF16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)p)[at] << 16);
    else return (float)((const _Float16*)p)[at];
}

template <int DT>
__device__ __forceinline__ void bal_store(void* p, size_t at, float v)
{
    if constexpr (DT == EVAMX_DTYPE_F32) {
        ((float*)p)[at] = v;
    } else if constexpr (DT == EVAMX_DTYPE_BF16) {
        uint32_t b = __builtin_bit_cast(uint32_t, v);
        b = (b & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : b + 0x7fffu + ((b >> 16) & 1);
        ((uint16_t*)p)[at] = (uint16_t)(b >> 16);
    } else {
        ((_Float16*)p)[at] = (_Float16)v;
    }
}

// Start of sequence s within the rows, whatever the table holds.
__device__ __forceinline__ int bal_start(const BalanceParams& p, int s)
{
    if (!p.starts) return s ? p.rows : 0;
    const int v = p.starts[s];
    return v < 0 ? 0 : v > p.rows ? p.rows : v;
}

// The sequence that holds a row: the last that starts at or before it (-1 before the first, `sequences` behind the last). Each
// step's 64 probes leave a 64th of the table.
__device__ __forceinline__ int bal_sequence(const BalanceParams& p, int row)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.sequences + 1;                          // starts[lo .. lo + n) hold the first one past the row
    while (n > 0) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const bool past = at >= lo + n || bal_start(p, at) > row;
        const unsigned long long b = __ballot(past);
        const int first = b ? __builtin_ctzll(b) : 64;        // probes before it start at or before the row
        if (first == 0) break;
        const int next = lo + (first - 1) * step + 1;
        n = (first - 1) * step + step < n ? step - 1 : n - (next - lo);
        lo = next;
    }
    return lo - 1;
}

// Sum over a wave in a fixed order, the same in every lane.
__device__ __forceinline__ float bal_wave_sum(float v)
{
    auto step = [](float a, auto ctrl) {
        return a + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, a), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    v = step(v, std::integral_constant<int, 0xb1>());         // lane ^ 1
    v = step(v, std::integral_constant<int, 0x4e>());         // lane ^ 2
    v = step(v, std::integral_constant<int, 0x141>());        // the half row mirrored
    v = step(v, std::integral_constant<int, 0x140>());        // the row of 16 mirrored
    const int b = __builtin_bit_cast(int, v);
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0)), r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
    const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32)), r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
    return (r0 + r1) + (r2 + r3);
}

// log(1 + e) for e in [0, 1], to a few fp32 steps: log(u) e / (u - 1) with u = 1 + e as rounded, whose error in u cancels.
__device__ __forceinline__ float bal_log1p(float e)
{
    const float u = 1.0f + e, d = u - 1.0f;
    return d == 0.0f ? e : __logf(u) * (e * __builtin_amdgcn_rcpf(d));
}

// The score of a logit and d log(score) / dz, by the hardware's exp2, log2, reciprocal and root (about one fp32 step each).
__device__ __forceinline__ void bal_score(float z, int score, float& a, float& slope)
{
    const float e = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    const float up = z >= 0 ? r : er, down = z >= 0 ? er : r;                       // sigma(z), sigma(-z)
    if (score == EVAMX_SCORE_SIGMOID) {
        a = up;
        slope = down;
    } else {
        const float sp = fmaxf(z, 0.0f) + bal_log1p(e);
        a = __builtin_amdgcn_sqrtf(sp);
        slope = z < -16.0f ? 0.5f : 0.5f * up * __builtin_amdgcn_rcpf(sp);           // 1 - e^z / 4 ..
    }
}

// The same for a row whose scores may all underflow: times 2^(lift / ln 2) (its root), which drops out of the shares, with the
// limit of the slope far below zero.
__device__ __forceinline__ float bal_score_far(float z, float lift, int score, float& slope)
{
    const float e = expf(-fabsf(z)), d = 1.0f / (1.0f + e);
    if (score == EVAMX_SCORE_SIGMOID) {
        slope = z >= 0 ? e * d : d;
        return z >= 0 ? d : expf(z + lift) * d;
    }
    const float sp = fmaxf(z, 0.0f) + log1pf(e);
    slope = z < -16.0f ? 0.5f : 0.5f * (z >= 0 ? d : e * d) / sp;
    return z < -16.0f ? expf(0.5f * (z + lift)) : sqrtf(sp) * expf(0.5f * lift);     // softplus(z) = e^z (1 - e^z / 2 ..)
}

// The shares of a row and the slopes, expert lane + 64 i in element i; z: the row's logits, -inf past the experts. A row whose
// logits are all -inf has none (zeros). Scores that underflow beside a sum over the threshold are below 2^-26 of it; smaller
// sums are made again relative to the row's largest logit.
template <int N>
__device__ __forceinline__ void bal_shares(const float (&z)[N], int score, float (&p)[N], float (&slope)[N])
{
    float sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        bal_score(z[i], score, p[i], slope[i]);
        sum += p[i];
    }
    sum = bal_wave_sum(sum);
    float inv = __builtin_amdgcn_rcpf(sum);
    if (!(sum >= (score == EVAMX_SCORE_SIGMOID ? 1e-30f : 1e-11f))) {
        const float inf = __builtin_inff();
        float top = -inf;
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, z[i]);
        for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
        const float lift = top < 0 && top > -inf ? -top : 0.0f;
        sum = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = bal_score_far(z[i], lift, score, slope[i]);
            sum += p[i];
        }
        sum = bal_wave_sum(sum);
        inv = top == -inf && sum == 0 ? 0.0f : 1.0f / sum;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] *= inv;
}

template <int N, int DT>
__device__ __forceinline__ void bal_row(const BalanceParams& q, int row, float (&z)[N])
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 64 * i;
        z[i] = e < q.experts ? bal_load<DT>(q.logits, row * q.stride + e) : -__builtin_inff();
    }
}

constexpr int BAL_WAVES = 8;
constexpr int bal_ahead(int n) { return n <= 4 ? 4 : 2; }     // rows a wave has on the way

// Sums of a chunk, one piece for each sequence that it meets: a wave takes a few rows at a time, a lane its experts' shares in
// registers; the waves meet in LDS in a fixed order, the picks are counted there (whole numbers: any order). 65536 x 256 logits in
// 24 sequences: 24.1 us, 3.0 TB/s of logits and picks; each value chooses the score function (built for sigmoid alone 21.1), and the
// next rows are requested when the present ones are summed.
template <int N, int DT>
__global__ __launch_bounds__(64 * BAL_WAVES) void balance_kernel(BalanceParams q)
{
    constexpr int BAL_AHEAD = bal_ahead(N);
    __shared__ float share[BAL_WAVES][64 * N];
    __shared__ int picks[64 * N], total;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = blockIdx.x * q.chunk, r1 = r0 + q.chunk < q.rows ? r0 + q.chunk : q.rows;
    if (blockIdx.x == 0)                                     // sequences that hold no row at all leave their words at rest
        for (int s = threadIdx.x; s < q.sequences; s += 64 * BAL_WAVES) q.arrive[(size_t)s * ARRIVE_STRIDE] = (unsigned long long)ARRIVE_REST << 32;
    for (int s = bal_sequence(q, r0), at = r0; at < r1;) {
        if (s >= q.sequences) break;
        int end = bal_start(q, s + 1);                       // of the rows before the first sequence too (s = -1)
        if (s < 0 || end <= at) {
            at = s < 0 ? end : at;
            ++s;
            continue;
        }
        if (end > r1) end = r1;
        for (int e = threadIdx.x; e < 64 * N; e += 64 * BAL_WAVES) picks[e] = 0;
        if (threadIdx.x == 0) total = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < (end - at) * q.topk; i += 64 * BAL_WAVES) {
            const int t = at + (q.topk == 1 ? i : (int)__umulhi((uint32_t)i, q.recip));
            const int64_t e = q.sel[(size_t)at * q.topk + i];
            if (e >= 0 && e < q.experts && (!q.mask || q.mask[t])) atomicAdd(&picks[e], 1);
        }
        float acc[N] = {};
        int n = 0;
        for (int t = at + wave * BAL_AHEAD; t < end; t += BAL_WAVES * BAL_AHEAD) {
            float z[BAL_AHEAD][N];
            bool use[BAL_AHEAD];
#pragma unroll
            for (int a = 0; a < BAL_AHEAD; ++a) {
                use[a] = t + a < end && (!q.mask || q.mask[t + a]);
                if (use[a]) bal_row<N, DT>(q, t + a, z[a]);
            }
#pragma unroll
            for (int a = 0; a < BAL_AHEAD; ++a) {
                if (!use[a]) continue;
                ++n;
                float p[N], slope[N];
                bal_shares<N>(z[a], q.score, p, slope);
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += p[i];
            }
        }
        if (lane == 0 && n) atomicAdd(&total, n);
#pragma unroll
        for (int i = 0; i < N; ++i) share[wave][lane + 64 * i] = acc[i];
        __syncthreads();
        const size_t piece = (size_t)blockIdx.x + s;
        for (int e = threadIdx.x; e < q.experts; e += 64 * BAL_WAVES) {
            float v = 0;
#pragma unroll
            for (int w = 0; w < BAL_WAVES; ++w) v += share[w][e];
            q.share[piece * q.experts + e] = v;
            q.picks[piece * q.experts + e] = picks[e];
        }
        if (threadIdx.x == 0) q.piece_tokens[piece] = total;
        __syncthreads();
        at = end;
        ++s;
    }
}

// Joins the pieces of a sequence: one workgroup for 64 of its experts, BAL_JOIN lanes an expert over the pieces. The last workgroup
// of a sequence to arrive adds the groups' products of picks and shares in order. 6.2 us for those 512 chunks (latency).
constexpr int BAL_JOIN = 16;

__global__ __launch_bounds__(64 * BAL_JOIN) void balance_join_kernel(BalanceParams q)
{
    __shared__ float share[BAL_JOIN][64];
    __shared__ int picks[BAL_JOIN][64], tok[BAL_JOIN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.x, groups = gridDim.y, e = 64 * blockIdx.y + lane;
    const int t0 = bal_start(q, s), t1 = bal_start(q, s + 1), w0 = t0 / q.chunk, w1 = t1 > t0 ? (t1 - 1) / q.chunk + 1 : w0;
    float p = 0;
    int c = 0, n = 0;
#pragma unroll 4
    for (int w = w0 + wave; w < w1; w += BAL_JOIN) {
        const size_t piece = (size_t)w + s;
        if (e < q.experts) {
            p += q.share[piece * q.experts + e];
            c += q.picks[piece * q.experts + e];
        }
        n += q.piece_tokens[piece];
    }
    share[wave][lane] = p;
    picks[wave][lane] = c;
    if (lane == 0) tok[wave] = n;
    __syncthreads();
    if (wave) return;
    p = 0;
    c = n = 0;
    for (int w = 0; w < BAL_JOIN; ++w) {
        p += share[w][lane];
        c += picks[w][lane];
        n += tok[w];
    }
    if (e < q.experts) q.counts[(size_t)s * q.experts + e] = c;
    const float part = bal_wave_sum((float)c * p), k = n ? (float)q.experts / ((float)q.topk * (float)n * (float)n) : 0.0f;
    if (blockIdx.y == 0 && lane == 0) q.tokens[s] = n;
    if (groups == 1) {
        if (lane == 0) q.loss[s] = k * part;
        return;
    }
    float* out = q.group_loss + (size_t)s * groups;
    if (lane == 0) __hip_atomic_store(out + blockIdx.y, part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!wave_arrive_last(q.arrive + (size_t)s * ARRIVE_STRIDE, (unsigned)groups)) return;
    float v = 0;
    for (int g = 0; g < groups; ++g) v += __hip_atomic_load(out + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (lane == 0) q.loss[s] = k * v;
}

// The gradient of a chunk's rows; a wave keeps the counts of the sequence it is in. Rows of no sequence, or masked, get zeros. The
// shares are made again from the logits: keeping them would write and read as many bytes as reading the logits again. 33 us for
// those logits, 4.0 TB/s read and written.
template <int N, int DT>
__global__ __launch_bounds__(64 * BAL_WAVES) void balance_grad_kernel(BalanceParams q)
{
    constexpr int BAL_AHEAD = bal_ahead(N);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = blockIdx.x * q.chunk, r1 = r0 + q.chunk < q.rows ? r0 + q.chunk : q.rows;
    for (int s = bal_sequence(q, r0), at = r0; at < r1;) {
        int end = s >= q.sequences ? r1 : bal_start(q, s + 1);
        if (end <= at) {
            ++s;
            continue;
        }
        if (end > r1) end = r1;
        const bool in = s >= 0 && s < q.sequences;
        float c[N] = {}, k = 0;
        if (in) {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = lane + 64 * i < q.experts ? (float)q.counts[(size_t)s * q.experts + lane + 64 * i] : 0.0f;
            const float n = (float)q.tokens[s];
            k = q.grad_loss[s] * ((float)q.experts / ((float)q.topk * n * n));
        }
        for (int t = at + wave * BAL_AHEAD; t < end; t += BAL_WAVES * BAL_AHEAD) {
            float z[BAL_AHEAD][N];
            bool use[BAL_AHEAD];
#pragma unroll
            for (int a = 0; a < BAL_AHEAD; ++a) {
                use[a] = in && t + a < end && (!q.mask || q.mask[t + a]);
                if (use[a]) bal_row<N, DT>(q, t + a, z[a]);
            }
#pragma unroll
            for (int a = 0; a < BAL_AHEAD; ++a) {
                if (t + a >= end) continue;
                float g[N] = {};
                if (use[a]) {
                    float p[N], slope[N], dot = 0;
                    bal_shares<N>(z[a], q.score, p, slope);
#pragma unroll
                    for (int i = 0; i < N; ++i) dot += c[i] * p[i];
                    dot = bal_wave_sum(dot);
#pragma unroll
                    for (int i = 0; i < N; ++i) g[i] = k * p[i] * (c[i] - dot) * slope[i];
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int e = lane + 64 * i;
                    if (e < q.experts) bal_store<DT>(q.grad, (size_t)(t + a) * q.experts + e, g[i]);
                }
            }
        }
        at = end;
        ++s;
    }
}

// f(experts per lane, dtype) with both as types.
template <class F>
static void balance_dispatch(const BalanceParams& p, F f)
{
    using std::integral_constant;
    auto type = [&](auto n) {
        if (p.dtype == EVAMX_DTYPE_F32) f(n, integral_constant<int, EVAMX_DTYPE_F32>());
        else if (p.dtype == EVAMX_DTYPE_BF16) f(n, integral_constant<int, EVAMX_DTYPE_BF16>());
        else f(n, integral_constant<int, EVAMX_DTYPE_F16>());
    };
    if (p.experts <= 64) type(integral_constant<int, 1>());
    else if (p.experts <= 128) type(integral_constant<int, 2>());
    else if (p.experts <= 256) type(integral_constant<int, 4>());
    else if (p.experts <= 384) type(integral_constant<int, 6>());
    else type(integral_constant<int, 8>());
}

// Rows of a chunk: enough workgroups to fill the GPU twice, few enough that their pieces are quickly joined.
static int balance_chunk(int rows)
{
    const int c = (rows + 511) / 512;
    return c < 32 ? 32 : c;
}

static size_t balance_align(size_t v) { return (v + 255) & ~(size_t)255; }

struct BalanceLayout {
    size_t share, picks, tokens, group_loss, arrive, total;
};

static BalanceLayout balance_layout(int rows, int experts, int sequences)
{
    const int chunk = balance_chunk(rows);
    const size_t pieces = (size_t)(rows + chunk - 1) / chunk + sequences;
    BalanceLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += balance_align(bytes); return o; };
    l.share = take(pieces * experts * 4);
    l.picks = take(pieces * experts * 4);
    l.tokens = take(pieces * 4);
    l.group_loss = take((size_t)sequences * ((experts + 63) / 64) * 4);
    l.arrive = take((size_t)sequences * ARRIVE_STRIDE * 8);
    l.total = at;
    return l;
}

}  // namespace evamx

using namespace evamx;

static bool balance_ok(const BalanceParams& p, const char* who)
{
    auto bad = [&](const char* what, long v) { set_error("%s: %s (%ld)", who, what, v); return false; };
    if (p.rows < 0 || p.rows > EVAMX_BALANCE_MAX_ROWS) return bad("rows outside 0..EVAMX_BALANCE_MAX_ROWS", p.rows);
    if (p.sequences < 1 || p.sequences > EVAMX_BALANCE_MAX_SEQUENCES) return bad("sequences outside 1..EVAMX_BALANCE_MAX_SEQUENCES", p.sequences);
    if (p.experts < 1 || p.experts > BAL_MAX_EXPERTS) return bad("experts outside 1..512", p.experts);
    if (p.topk < 1 || p.topk > 32) return bad("topk outside 1..32", p.topk);
    if (p.score != EVAMX_SCORE_SIGMOID && p.score != EVAMX_SCORE_SQRT_SOFTPLUS) return bad("unknown score function", p.score);
    if (p.dtype != EVAMX_DTYPE_F16 && p.dtype != EVAMX_DTYPE_BF16 && p.dtype != EVAMX_DTYPE_F32) return bad("unknown dtype", p.dtype);
    if (p.stride < (size_t)p.experts || p.stride > ((size_t)1 << 40)) return bad("row stride below the experts", (long)p.stride);
    if ((!p.logits || !p.sel) && p.rows) return bad("null logits or sel", 0);
    if (!p.starts && p.sequences != 1) return bad("several sequences need their starts", p.sequences);
    if (!p.counts || !p.tokens) return bad("null counts or tokens", 0);
    return true;
}

static BalanceParams balance_params(const void* logits, int dtype, int64_t stride, int rows, int experts, const int64_t* sel, int topk,
                                    int score_fn, const int32_t* starts, int sequences, const uint8_t* mask)
{
    BalanceParams p;
    memset(&p, 0, sizeof p);
    p.logits = logits; p.dtype = dtype; p.stride = stride < 0 ? 0 : (size_t)stride; p.rows = rows; p.experts = experts;
    p.chunk = balance_chunk(rows); p.recip = topk > 0 ? (uint32_t)(((1ull << 32) + topk - 1) / topk) : 0;
    p.sel = sel; p.topk = topk; p.score = score_fn; p.starts = starts; p.sequences = sequences; p.mask = mask;
    return p;
}

extern "C" size_t evamx_balance_workspace_bytes(int rows, int experts, int sequences)
{
    if (rows < 0 || rows > EVAMX_BALANCE_MAX_ROWS || experts < 1 || experts > BAL_MAX_EXPERTS || sequences < 1 ||
        sequences > EVAMX_BALANCE_MAX_SEQUENCES)
        return 0;
    return balance_layout(rows, experts, sequences).total;
}

extern "C" int evamx_balance_loss(const void* logits, int dtype, int64_t stride, int rows, int experts, const int64_t* sel, int topk,
                                  int score_fn, const int32_t* starts, int sequences, const uint8_t* mask, float* loss, int32_t* counts,
                                  int32_t* tokens, void* workspace, size_t workspace_bytes, evamx_stream_t stream)
{
    set_error("%s", "");
    BalanceParams p = balance_params(logits, dtype, stride, rows, experts, sel, topk, score_fn, starts, sequences, mask);
    p.loss = loss; p.counts = counts; p.tokens = tokens;
    if (!balance_ok(p, "evamx_balance_loss")) return EVAMX_EINVAL;
    if ((uintptr_t)workspace & 15) { set_error("evamx_balance_loss: the workspace must be 16-byte aligned"); return EVAMX_EINVAL; }
    if (!loss || !workspace) { set_error("evamx_balance_loss: null pointer"); return EVAMX_EINVAL; }
    const size_t need = evamx_balance_workspace_bytes(rows, experts, sequences);
    if (workspace_bytes < need) { set_error("evamx_balance_loss: workspace %zu bytes < %zu", workspace_bytes, need); return EVAMX_ENOSPACE; }
    char* ws = (char*)workspace;
    const BalanceLayout l = balance_layout(rows, experts, sequences);
    p.share = (float*)(ws + l.share); p.picks = (int32_t*)(ws + l.picks); p.piece_tokens = (int32_t*)(ws + l.tokens);
    p.group_loss = (float*)(ws + l.group_loss); p.arrive = (unsigned long long*)(ws + l.arrive);
    const int chunks = rows ? (rows + p.chunk - 1) / p.chunk : 1;
    balance_dispatch(p, [&](auto n, auto dt) {
        balance_kernel<decltype(n)::value, decltype(dt)::value><<<chunks, 64 * BAL_WAVES, 0, (hipStream_t)stream>>>(p);
    });
    balance_join_kernel<<<dim3(sequences, (experts + 63) / 64), 64 * BAL_JOIN, 0, (hipStream_t)stream>>>(p);
    return launched("balance_loss");
}

extern "C" int evamx_balance_grad(const float* grad_loss, const void* logits, int dtype, int64_t stride, int rows, int experts,
                                  int topk, int score_fn, const int32_t* starts, int sequences, const uint8_t* mask,
                                  const int32_t* counts, const int32_t* tokens, void* grad, evamx_stream_t stream)
{
    set_error("%s", "");
    BalanceParams p = balance_params(logits, dtype, stride, rows, experts, (const int64_t*)logits, topk, score_fn, starts, sequences, mask);
    p.counts = const_cast<int32_t*>(counts); p.tokens = const_cast<int32_t*>(tokens);
    p.grad_loss = grad_loss; p.grad = grad;
    if (!balance_ok(p, "evamx_balance_grad")) return EVAMX_EINVAL;
    if (!grad_loss || (!grad && rows)) { set_error("evamx_balance_grad: null pointer"); return EVAMX_EINVAL; }
    if (rows == 0) return EVAMX_OK;
    balance_dispatch(p, [&](auto n, auto dt) {
        balance_grad_kernel<decltype(n)::value, decltype(dt)::value><<<(rows + p.chunk - 1) / p.chunk, 64 * BAL_WAVES, 0, (hipStream_t)stream>>>(p);
    });
    return launched("balance_grad");
}
