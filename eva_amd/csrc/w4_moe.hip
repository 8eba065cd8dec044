// The routed (and shared) SwiGLU experts of an MoE layer on 4-bit weights with group scales (w4.hpp):
//   out[t] = sum_k w_tk D_e h_tk,  h = min(silu(G_e x_t), L) * clamp(U_e x_t, -L, L),  e = sel[t][k] - first_expert,
// over the slots whose e lies in [0, n_local); the shared experts are the last matrices of the stacks, weight 1, every token,
// their gate clamped before SiLU (both as evamx_moe_forward has them). L = 0: no clamping.
#include <cmath>

#include "evamx_internal.hpp"
#include "w4.hpp"

namespace evamx {

struct W4MoeParams {
    int rows, topk, n_shared, kt_slots, slots, n_local, count, hidden, inter, bf16;   // kt_slots = topk + n_shared per token
    long long first;
    float limit;
    const int64_t* sel;
    const float* weights;
    int* offsets;                // [count + 1]: positions of an expert's slots in `order`; the last is their number
    int* order;                  // [slots]: slots by (expert, slot)
    const w4_half* x;            // [rows][k of gate, padded], with a factor per row
    const float* xs;
    float* h;                    // [positions][inter]
    w4_half* hh;                 // the same, ready for the down products, with a factor per row
    float* hs;
    float* y;                    // [slots][hidden]
    void* out;
    size_t out_stride;
};

// Matrix of slot s, or -1.
__device__ __forceinline__ int w4_slot_expert(const W4MoeParams& p, int s)
{
    const int t = s / p.kt_slots, k = s - t * p.kt_slots;
    if (k >= p.topk) return p.n_local + k - p.topk;
    const unsigned long long e = (unsigned long long)p.sel[(size_t)t * p.topk + k] - (unsigned long long)p.first;    // wraps
    return e < (unsigned)p.n_local ? (int)e : -1;
}

// Stable grouping, one workgroup an expert: it counts the slots of smaller experts and its own, then writes its own in
// order. count x slots reads from L2, far below the products that follow.
__global__ __launch_bounds__(256) void w4_group_kernel(W4MoeParams p)
{
    __shared__ int part[4], wave_n[4];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int less = 0;
    for (int s = threadIdx.x; s < p.slots; s += 256) {
        const int v = w4_slot_expert(p, s);
        less += v >= 0 && v < e;
    }
    for (int i = 32; i; i >>= 1) less += __shfl_xor(less, i);
    if (lane == 0) part[wave] = less;
    __syncthreads();
    int at = part[0] + part[1] + part[2] + part[3];
    if (threadIdx.x == 0) p.offsets[e] = at;
    for (int s0 = 0; s0 < p.slots; s0 += 256) {
        const int s = s0 + threadIdx.x;
        const bool mine = s < p.slots && w4_slot_expert(p, s) == e;
        const unsigned long long b = __ballot(mine);
        if (lane == 0) wave_n[wave] = __popcll(b);
        __syncthreads();
        int pos = at + __popcll(b & ((1ull << lane) - 1));
        for (int w = 0; w < wave; ++w) pos += wave_n[w];
        if (mine) p.order[pos] = s;
        at += wave_n[0] + wave_n[1] + wave_n[2] + wave_n[3];
        __syncthreads();
    }
    if (e == p.count - 1 && threadIdx.x == 0) p.offsets[p.count] = at;
}

struct W4Unit {
    int expert, r0, rows;        // positions r0 .. r0 + rows - 1 of the order; expert -1: past the last unit
};

// The unit'th block of at most `tile` positions of one expert, found by every wave on its own.
__device__ __forceinline__ W4Unit w4_unit(const int* __restrict__ offsets, int count, int tile, int unit)
{
    const int lane = threadIdx.x & 63, per = (count + 63) / 64;
    int n = 0;
    for (int i = 0; i < per; ++i) {
        const int e = lane * per + i;
        if (e < count) n += (offsets[e + 1] - offsets[e] + tile - 1) / tile;
    }
    int incl = n;
    for (int s = 1; s < 64; s <<= 1) {
        const int v = __shfl_up(incl, s);
        if (lane >= s) incl += v;
    }
    const unsigned long long here = __ballot(incl > unit);
    if (!here) return {-1, 0, 0};
    const int owner = __builtin_ctzll(here);
    W4Unit u = {-1, 0, 0};
    if (lane == owner) {
        int left = unit - (incl - n);
        for (int i = 0; i < per; ++i) {
            const int e = lane * per + i;
            if (e >= count) break;
            const int o = offsets[e], c = offsets[e + 1] - o, t = (c + tile - 1) / tile;
            if (left < t) {
                u = {e, o + left * tile, c - left * tile < tile ? c - left * tile : tile};
                break;
            }
            left -= t;
        }
    }
    return {__shfl(u.expert, owner), __shfl(u.r0, owner), __shfl(u.rows, owner)};
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

// 16 columns of gate and up by 16 positions of one expert; the four waves take every fourth quad of k-tiles.
template <int SG, bool ZERO>
__global__ __launch_bounds__(256) void w4_gate_up_kernel(W4MoeParams p, W4Mat gate, W4Mat up)
{
    __shared__ w4_f32x4 part[4][2][64];
    const W4Unit u = w4_unit(p.offsets, p.count, 16, blockIdx.y);
    if (u.expert < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = blockIdx.x;
    const w4_half* a = nullptr;
    if ((lane & 15) < u.rows) {
        const int t = p.order[u.r0 + (lane & 15)] / p.kt_slots;
        a = p.x + (size_t)t * gate.kt * W4_TILE_K + 8 * (lane >> 4);
    }
    w4_f32x4 g = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    w4_accumulate<SG, ZERO>(g, gate, u.expert, nt, a, wave, 4);
    w4_accumulate<SG, ZERO>(v, up, u.expert, nt, a, wave, 4);
    part[wave][0][lane] = g;
    part[wave][1][lane] = v;
    __syncthreads();
    const int r = 4 * (lane >> 4) + wave, n = 16 * nt + (lane & 15);
    if (r >= u.rows || n >= p.inter) return;
    float gs = 0, us = 0;
    for (int w = 0; w < 4; ++w) {
        gs += part[w][0][lane][wave];
        us += part[w][1][lane][wave];
    }
    const float xs = p.xs[p.order[u.r0 + r] / p.kt_slots];
    p.h[(size_t)(u.r0 + r) * p.inter + n] = w4_swiglu(gs * xs, us * xs, p.limit, u.expert >= p.n_local);
}

// The hidden activations of the positions there are, ready for the down products (w4_rows_kernel's scheme).
__global__ __launch_bounds__(256) void w4_hidden_kernel(W4MoeParams p, int n_pad)
{
    __shared__ uint32_t part[4];
    if ((int)blockIdx.x >= p.offsets[p.count]) return;
    const float* row = p.h + (size_t)blockIdx.x * p.inter;
    uint32_t top = 0;
    for (int k = threadIdx.x; k < p.inter; k += 256) {
        const uint32_t b = __builtin_bit_cast(uint32_t, row[k]) & 0x7fffffffu;
        if (b < 0x7f800000u && b > top) top = b;
    }
    for (int s = 32; s; s >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, s);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < 4; ++i) top = part[i] > top ? part[i] : top;
    const int e = w4_exponent(top);
    const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    for (int k = threadIdx.x; k < n_pad; k += 256)
        p.hh[blockIdx.x * (size_t)n_pad + k] = k < p.inter ? (w4_half)(row[k] * down) : (w4_half)0.0f;
    if (threadIdx.x == 0) p.hs[blockIdx.x] = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
}

template <int SG, bool ZERO>
__global__ __launch_bounds__(256) void w4_down_kernel(W4MoeParams p, W4Mat down)
{
    __shared__ w4_f32x4 part[4][64];
    const W4Unit u = w4_unit(p.offsets, p.count, 16, blockIdx.y);
    if (u.expert < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = blockIdx.x;
    w4_f32x4 acc = {0, 0, 0, 0};
    w4_accumulate<SG, ZERO>(acc, down, u.expert, nt,
                            (lane & 15) < u.rows ? p.hh + (size_t)(u.r0 + (lane & 15)) * down.kt * W4_TILE_K + 8 * (lane >> 4) : nullptr, wave, 4);
    part[wave][lane] = acc;
    __syncthreads();
    const int r = 4 * (lane >> 4) + wave, n = 16 * nt + (lane & 15);
    if (r >= u.rows || n >= p.hidden) return;
    float v = 0;
    for (int w = 0; w < 4; ++w) v += part[w][lane][wave];
    p.y[(size_t)p.order[u.r0 + r] * p.hidden + n] = v * p.hs[u.r0 + r];
}

// out[t] = the slots' outputs in slot order times their routing weights (fp32, as given), rounded once.
__global__ __launch_bounds__(256) void w4_combine_kernel(W4MoeParams p)
{
    const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    if (n >= p.hidden) return;
    float v = 0;
    for (int k = 0; k < p.kt_slots; ++k) {
        const int s = t * p.kt_slots + k;
        if (w4_slot_expert(p, s) < 0) continue;
        v += (k < p.topk ? p.weights[(size_t)t * p.topk + k] : 1.0f) * p.y[(size_t)s * p.hidden + n];
    }
    w4_store(p.out, (size_t)t * p.out_stride + n, v, p.bf16);
}

struct W4MoeLayout {
    size_t offsets, order, xs, x, h, hs, hh, y, total;
};

static W4MoeLayout w4_moe_layout(int rows, int topk, int n_shared, int hidden, int inter)
{
    const size_t slots = (size_t)rows * (topk + n_shared);
    const size_t kx = (size_t)w4_ceil(hidden, W4_TILE_K) * W4_TILE_K, kh = (size_t)w4_ceil(inter, W4_TILE_K) * W4_TILE_K;
    W4MoeLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += w4_align(bytes); return o; };
    l.offsets = take(1025 * 4);
    l.order = take(slots * 4);
    l.xs = take((size_t)rows * 4);
    l.x = take(rows * kx * 2);
    l.h = take(slots * inter * 4);
    l.hs = take(slots * 4);
    l.hh = take(slots * kh * 2);
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
    return true;
}

template <int SG, bool ZERO>
static void w4_launch_gate_up(const W4MoeParams& p, const W4Mat& gate, const W4Mat& up, int units, hipStream_t s)
{
    w4_gate_up_kernel<SG, ZERO><<<dim3(w4_ceil(p.inter, 16), units), 256, 0, s>>>(p, gate, up);
}

template <int SG, bool ZERO>
static void w4_launch_down(const W4MoeParams& p, const W4Mat& down, int units, hipStream_t s)
{
    w4_down_kernel<SG, ZERO><<<dim3(w4_ceil(p.hidden, 16), units), 256, 0, s>>>(p, down);
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
    if (g.group != u.group || (g.zeros == nullptr) != (u.zeros == nullptr)) {
        set_error("%s: gate and up differ in their group size or zero points", who);
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
    p.first = a->first_expert; p.limit = a->limit; p.sel = a->sel; p.weights = a->weights;
    p.offsets = (int*)(ws + l.offsets); p.order = (int*)(ws + l.order);
    p.x = (const w4_half*)(ws + l.x); p.xs = (const float*)(ws + l.xs);
    p.h = (float*)(ws + l.h); p.hh = (w4_half*)(ws + l.hh); p.hs = (float*)(ws + l.hs); p.y = (float*)(ws + l.y);
    p.out = a->out; p.out_stride = (size_t)a->out_stride;
    const hipStream_t s = (hipStream_t)stream;
    const W4Mat gm = w4_mat(g), um = w4_mat(u), dm = w4_mat(d);
    const int units = (p.slots < p.count ? p.slots : p.count) + p.slots / 16;

    w4_launch_rows(a->x, a->x_dtype, (size_t)a->x_stride, p.rows, p.hidden, ws + l.x, (float*)(ws + l.xs), s);
    w4_group_kernel<<<p.count, 256, 0, s>>>(p);
    w4_dispatch(g, [&](auto sg, auto zero) { w4_launch_gate_up<decltype(sg)::value, decltype(zero)::value>(p, gm, um, units, s); });
    w4_hidden_kernel<<<p.slots, 256, 0, s>>>(p, dm.kt * W4_TILE_K);
    w4_dispatch(d, [&](auto sg, auto zero) { w4_launch_down<decltype(sg)::value, decltype(zero)::value>(p, dm, units, s); });
    w4_combine_kernel<<<dim3(w4_ceil(p.hidden, 256), p.rows), 256, 0, s>>>(p);
    return launched("w4_moe_forward");
}
