// Per-sequence expert counts and balance loss of a router, and the loss's gradient.
//
// Token t of sequence s has scores a_e = score(z_te) (the router's score function), shares p_e = a_e / sum a and topk picks
// sel. With n valid tokens and c_e picks of expert e in the sequence,
//   L_s = sum_e f_e P_e,  f_e = E c_e / (topk n),  P_e = (1/n) sum_t p_te       (1 where picks and shares are even).
// The counts are constants of the gradient:
//   dL_s/dz_tj = E / (topk n^2) * p_tj * (c_j - sum_i c_i p_ti) * dlog a_j/dz_j,
//   dlog a/dz = sigma(-z) for sigmoid, sigma(z) / (2 softplus(z)) for sqrt(softplus).
#include <cstring>

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
};

__device__ __forceinline__ float bal_load(const void* p, size_t at, int dtype)
{
    if (dtype == EVAMX_DTYPE_F32) return ((const float*)p)[at];
    if (dtype == EVAMX_DTYPE_BF16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)p)[at] << 16);
    return (float)((const _Float16*)p)[at];
}

__device__ __forceinline__ void bal_store(void* p, size_t at, float v, int dtype)
{
    if (dtype == EVAMX_DTYPE_F32) {
        ((float*)p)[at] = v;
    } else if (dtype == EVAMX_DTYPE_BF16) {
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

// score(z) * 2^(shift): the row's shift lifts rows whose scores would all underflow; it drops out of the shares.
__device__ __forceinline__ float bal_score(float z, float lift, int score)
{
    const float e = expf(-fabsf(z));                                     // in (0, 1]; 0 at infinity
    if (score == EVAMX_SCORE_SIGMOID) return z >= 0 ? 1.0f / (1.0f + e) : expf(z + lift) / (1.0f + e);
    if (z >= -16.0f) return sqrtf(fmaxf(z, 0.0f) + log1pf(e)) * expf(0.5f * lift);
    return expf(0.5f * (z + lift));                                      // softplus(z) = e^z (1 - e^z / 2 ..)
}

__device__ __forceinline__ float bal_slope(float z, int score)
{
    const float e = expf(-fabsf(z)), d = 1.0f / (1.0f + e);
    if (score == EVAMX_SCORE_SIGMOID) return z >= 0 ? e * d : d;
    if (z < -16.0f) return 0.5f;
    return 0.5f * (z >= 0 ? d : e * d) / (fmaxf(z, 0.0f) + log1pf(e));
}

template <class T, class F>
__device__ __forceinline__ T wave_all(T v, F f)
{
    for (int s = 32; s; s >>= 1) v = f(v, __shfl_xor(v, s));
    return v;
}

// The row's shares in a wave's lanes: p[i] is expert lane + 64 i. A row whose logits are all -inf has none (zeros).
__device__ __forceinline__ void bal_shares(const BalanceParams& q, int row, float (&z)[BAL_MAX_EXPERTS / 64], float (&p)[BAL_MAX_EXPERTS / 64])
{
    const int lane = threadIdx.x & 63;
    const float inf = __builtin_inff();
    float top = -inf;
#pragma unroll
    for (int i = 0; i < BAL_MAX_EXPERTS / 64; ++i) {
        const int e = lane + 64 * i;
        z[i] = e < q.experts ? bal_load(q.logits, row * q.stride + e, q.dtype) : -inf;
        top = fmaxf(top, z[i]);
    }
    top = wave_all(top, [](float a, float b) { return fmaxf(a, b); });
    const float lift = top < 0 && top > -inf ? -top : 0.0f;
    float sum = 0;
#pragma unroll
    for (int i = 0; i < BAL_MAX_EXPERTS / 64; ++i) {
        p[i] = bal_score(z[i], lift, q.score);
        sum += p[i];
    }
    sum = wave_all(sum, [](float a, float b) { return a + b; });
    const float inv = top == -inf && sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < BAL_MAX_EXPERTS / 64; ++i) p[i] *= inv;
}

// One workgroup a sequence: its four waves take every fourth token, their sums meet in LDS in a fixed order.
__global__ __launch_bounds__(256) void balance_kernel(BalanceParams q)
{
    constexpr int N = BAL_MAX_EXPERTS / 64;
    __shared__ float share[4][BAL_MAX_EXPERTS];
    __shared__ int picks[BAL_MAX_EXPERTS], total;
    __shared__ float part[4];
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < BAL_MAX_EXPERTS; e += 256) picks[e] = 0;
    if (threadIdx.x == 0) total = 0;
    __syncthreads();
    const int t0 = bal_start(q, s), t1 = bal_start(q, s + 1);
    float acc[N] = {};
    int n = 0;
    for (int t = t0 + wave; t < t1; t += 4) {
        if (q.mask && !q.mask[t]) continue;
        ++n;
        float z[N], p[N];
        bal_shares(q, t, z, p);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += p[i];
        if (lane < q.topk) {
            const int64_t e = q.sel[(size_t)t * q.topk + lane];
            if (e >= 0 && e < q.experts) atomicAdd(&picks[e], 1);
        }
    }
    if (lane == 0 && n) atomicAdd(&total, n);
#pragma unroll
    for (int i = 0; i < N; ++i) share[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    float v = 0;
    for (int e = threadIdx.x; e < q.experts; e += 256) {
        v += (float)picks[e] * ((share[0][e] + share[1][e]) + (share[2][e] + share[3][e]));
        q.counts[(size_t)s * q.experts + e] = picks[e];
    }
    v = wave_all(v, [](float a, float b) { return a + b; });
    if (lane == 0) part[wave] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        const float k = total ? (float)q.experts / ((float)q.topk * (float)total * (float)total) : 0.0f;
        q.loss[s] = k * ((part[0] + part[1]) + (part[2] + part[3]));
        q.tokens[s] = total;
    }
}

// One wave a row. A row of no sequence, or masked, has a zero gradient.
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceParams q)
{
    constexpr int N = BAL_MAX_EXPERTS / 64;
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= q.rows) return;
    int s = -1;
    if (!q.mask || q.mask[t])
        for (int i = 0; i < q.sequences; ++i)
            if (t >= bal_start(q, i) && t < bal_start(q, i + 1)) s = i;
    float g[N] = {};
    if (s >= 0) {
        float z[N], p[N], c[N], dot = 0;
        bal_shares(q, t, z, p);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 64 * i;
            c[i] = e < q.experts ? (float)q.counts[(size_t)s * q.experts + e] : 0.0f;
            dot += c[i] * p[i];
        }
        dot = wave_all(dot, [](float a, float b) { return a + b; });
        const float n = (float)q.tokens[s], k = q.grad_loss[s] * ((float)q.experts / ((float)q.topk * n * n));
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = k * p[i] * (c[i] - dot) * bal_slope(z[i], q.score);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 64 * i;
        if (e < q.experts) bal_store(q.grad, (size_t)t * q.experts + e, g[i], q.dtype);
    }
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
    p.sel = sel; p.topk = topk; p.score = score_fn; p.starts = starts; p.sequences = sequences; p.mask = mask;
    return p;
}

extern "C" size_t evamx_balance_workspace_bytes(int rows, int experts, int sequences)
{
    return 256;
}

extern "C" int evamx_balance_loss(const void* logits, int dtype, int64_t stride, int rows, int experts, const int64_t* sel, int topk,
                                  int score_fn, const int32_t* starts, int sequences, const uint8_t* mask, float* loss, int32_t* counts,
                                  int32_t* tokens, void* workspace, size_t workspace_bytes, evamx_stream_t stream)
{
    set_error("%s", "");
    BalanceParams p = balance_params(logits, dtype, stride, rows, experts, sel, topk, score_fn, starts, sequences, mask);
    p.loss = loss; p.counts = counts; p.tokens = tokens;
    if (!balance_ok(p, "evamx_balance_loss")) return EVAMX_EINVAL;
    if (!loss || !workspace) { set_error("evamx_balance_loss: null pointer"); return EVAMX_EINVAL; }
    const size_t need = evamx_balance_workspace_bytes(rows, experts, sequences);
    if (workspace_bytes < need) { set_error("evamx_balance_loss: workspace %zu bytes < %zu", workspace_bytes, need); return EVAMX_ENOSPACE; }
    balance_kernel<<<sequences, 256, 0, (hipStream_t)stream>>>(p);
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
    balance_grad_kernel<<<(rows + 3) / 4, 256, 0, (hipStream_t)stream>>>(p);
    return launched("balance_grad");
}
