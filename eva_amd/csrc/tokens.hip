// Tokens sorted by expert and back: the order, the sorted rows, their weighted sums, and the gradients of both.
//
// Slot (t, k) of token t takes expert e = sel[t][k] - first. Rows are sorted by expert, an expert's in the order of its slots:
//   position[t][k] = starts[e] + #{slots of e before (t, k)},   -1 for a slot of no local expert,
//   sorted rows      s[position[t][k]] = x[t]                   (gradient: the sum below with weights of 1),
//   weighted sums    out[t] = sum_k w[t][k] y[position[t][k]] + residual[t],
//   their gradients  dy[position[t][k]] = w[t][k] g[t],  dw[t][k] = <g[t], y[position[t][k]]>.
// Rows behind starts[n_local] belong to no slot and are zeros. Every kernel here is bound by memory: a token's row is read once
// and written topk times, or the other way round.
#include <type_traits>

#include "evamx_gemv.hpp"
#include "evamx_internal.hpp"

namespace evamx {

constexpr int TOK_MAX_EXPERTS = 1024, TOK_MAX_TOPK = 32;
constexpr int64_t TOK_MAX_SLOTS = 1 << 26;

// ---- the order ---------------------------------------------------------------------------------

// Chunks of consecutive slots, a workgroup each; a workgroup's waves take consecutive segments of it. Up to 2048 slots one launch (8
// slots: 3.6 us, of which a launch is 1.6), more in two, whose second sums the first's counts again in every workgroup (131072 slots
// of 256 experts: 4.7 and 8.2 us).
constexpr int ORD_WAVES = 16, ORD_THREADS = 64 * ORD_WAVES, ORD_MAX_CHUNKS = 256;

struct OrderParams {
    const int64_t* sel;
    int64_t first;
    int slots, n_local, chunk, segment, chunks;
    int32_t* starts;
    int32_t* position;
    int32_t* counts;            // [chunks][n_local]
};

__device__ __forceinline__ int ord_expert(const OrderParams& p, int slot)
{
    const uint64_t e = (uint64_t)p.sel[slot] - (uint64_t)p.first;       // a difference past 64 bits wraps to no expert's number
    return e < (uint64_t)p.n_local && (p.sel[slot] >= p.first) ? (int)e : -1;
}

// The slots of a wave's segment: [lo, hi).
__device__ __forceinline__ void ord_segment(const OrderParams& p, int wave, int& lo, int& hi)
{
    const int64_t end = min((int64_t)p.slots, ((int64_t)blockIdx.x + 1) * p.chunk);
    const int64_t a = (int64_t)blockIdx.x * p.chunk + (int64_t)wave * p.segment;
    lo = (int)min(a, end);
    hi = (int)min(a + p.segment, end);
}

__global__ __launch_bounds__(ORD_THREADS) void order_count_kernel(OrderParams p)
{
    __shared__ int count[TOK_MAX_EXPERTS];
    for (int e = threadIdx.x; e < p.n_local; e += ORD_THREADS) count[e] = 0;
    __syncthreads();
    int lo, hi;
    ord_segment(p, threadIdx.x >> 6, lo, hi);
    for (int s = lo + (threadIdx.x & 63); s < hi; s += 64) {
        const int e = ord_expert(p, s);
        if (e >= 0) atomicAdd(&count[e], 1);                            // whole numbers: the order does not matter
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_local; e += ORD_THREADS) p.counts[(size_t)blockIdx.x * p.n_local + e] = count[e];
}

// Places the slots of a chunk. ONE: the only chunk, which counts by itself. 64 slots of a wave are ranked at once: lanes with the
// same expert find each other with a ballot for each bit of its number.
template <bool ONE>
__global__ __launch_bounds__(ORD_THREADS) void order_place_kernel(OrderParams p, int bits)
{
    extern __shared__ int seg[];                                        // [ORD_WAVES][n_local]: first counts, then the next places
    __shared__ int wave_sum[ORD_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < ORD_WAVES * p.n_local; i += ORD_THREADS) seg[i] = 0;
    __syncthreads();
    int lo, hi;
    ord_segment(p, wave, lo, hi);
    for (int s = lo + lane; s < hi; s += 64) {
        const int e = ord_expert(p, s);
        if (e >= 0) atomicAdd(&seg[wave * p.n_local + e], 1);
    }
    __syncthreads();
    // thread e: expert e's slots in all chunks and in those before this one
    const int e = threadIdx.x;
    int all = 0, before = 0;
    if (e < p.n_local) {
        if (ONE) {
            for (int w = 0; w < ORD_WAVES; ++w) all += seg[w * p.n_local + e];
        } else {
#pragma unroll 8
            for (int c = 0; c < p.chunks; ++c) {
                const int n = p.counts[(size_t)c * p.n_local + e];
                all += n;
                before += c < (int)blockIdx.x ? n : 0;
            }
        }
    }
    int upto = all;                                                     // inclusive sum over the experts
    for (int d = 1; d < 64; d <<= 1) {
        const int n = __shfl_up(upto, d);
        if (lane >= d) upto += n;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += wave_sum[w];
    if (e < p.n_local) {
        int at = upto - all;
        if (blockIdx.x == 0) {
            p.starts[e] = at;
            if (e == p.n_local - 1) p.starts[p.n_local] = upto;
        }
        at += before;
        for (int w = 0; w < ORD_WAVES; ++w) {
            const int n = seg[w * p.n_local + e];
            seg[w * p.n_local + e] = at;
            at += n;
        }
    }
    __syncthreads();
    int* next = seg + wave * p.n_local;
    for (int s0 = lo; s0 < hi; s0 += 64) {
        const int s = s0 + lane, x = s < hi ? ord_expert(p, s) : -1;
        unsigned long long same = __ballot(x >= 0);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(x >> b & 1);
            same &= (x >> b & 1) ? set : ~set;
        }
        const unsigned long long below = same & ((1ull << lane) - 1);
        int at = -1;
        if (x >= 0) at = next[x] + __popcll(below);
        wave_lds_fence();                                               // all have read before the last of each expert writes
        if (x >= 0 && (same >> lane) == 1) next[x] = at + 1;
        wave_lds_fence();
        if (s < hi) p.position[s] = at;
    }
}

// ---- rows --------------------------------------------------------------------------------------

// 16 bytes of a row at any alignment of its type: the hardware takes unaligned pieces, only slower.
template <int DT>
struct TokPiece {
    static constexpr int N = DT == EVAMX_DTYPE_F32 ? 4 : 8;            // values
    typedef typename std::conditional<DT == EVAMX_DTYPE_F32, float, uint16_t>::type type;
    typedef type vec __attribute__((ext_vector_type(N)));
    typedef vec loose __attribute__((aligned(sizeof(type))));
    vec v;

    // STREAM: what is not read again before the caches have lost it
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const void* p, size_t at, int have)
    {
        if (have >= N) {
            const loose* from = (const loose*)((const type*)p + at);
            if constexpr (STREAM) v = __builtin_nontemporal_load(from);
            else v = *from;
        } else {
            for (int i = 0; i < N; ++i) v[i] = i < have ? ((const type*)p)[at + i] : 0;
        }
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(void* p, size_t at, int have) const
    {
        if (have >= N) {
            loose* to = (loose*)((type*)p + at);
            if constexpr (STREAM) __builtin_nontemporal_store(v, to);
            else *to = v;
        } else {
            for (int i = 0; i < have; ++i) ((type*)p)[at + i] = v[i];
        }
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (DT == EVAMX_DTYPE_F32) return v[i];
        else if constexpr (DT == EVAMX_DTYPE_BF16) return __builtin_bit_cast(float, (uint32_t)v[i] << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)v[i]);
    }
    __device__ __forceinline__ void set(int i, float f)                // to nearest, ties to even; a NaN stays one
    {
        if constexpr (DT == EVAMX_DTYPE_F32) {
            v[i] = f;
        } else if constexpr (DT == EVAMX_DTYPE_BF16) {
            v[i] = __builtin_bit_cast(uint16_t, (__bf16)f);
        } else {
            v[i] = __builtin_bit_cast(uint16_t, (_Float16)f);
        }
    }
};

struct TokenParams {
    int rows, hidden, topk, n_local;
    const int32_t* position;
    const int32_t* starts;
    int64_t sorted_rows;
    const void* in;                              // x, or the sorted rows, or the sums' gradient
    size_t in_stride;
    const void* y;                               // the sorted rows of the sums whose gradient is taken
    size_t y_stride;
    const float* weights;
    const void* residual;
    size_t residual_stride;
    void* out;
    size_t out_stride;
    float* grad_weights;
};

// Workgroups of up to `most` waves: a row's parts, or a token's slots, over as few workgroups as that takes, evenly. Sums that
// stream take 16 (16384 tokens: 366 us, with 8 372), others 8 (16 tokens: 4.3 us, with 16 5.1).
constexpr int TOK_WAVES = 8, TOK_SUM_WAVES = 16;
struct TokGrid {
    int groups, waves;
    TokGrid(int units, int most) : groups((units + most - 1) / most), waves((units + groups - 1) / groups) {}
};

__device__ __forceinline__ int tok_unit() { return blockIdx.y * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Zeros in the sorted rows behind the last one that belongs to a slot, by the workgroups behind those of the tokens.
template <int DT, bool STREAM>
__device__ __forceinline__ void tok_zero_tail(const TokenParams& p)
{
    const int b = (blockIdx.x - p.rows) * gridDim.y + blockIdx.y, n = (gridDim.x - p.rows) * gridDim.y;
    int64_t r = p.starts[p.n_local];
    r = r < 0 ? 0 : r;
    TokPiece<DT> zero;
    zero.v = 0;
    for (r += b; r < p.sorted_rows; r += n)
        for (int c = threadIdx.x * zero.N; c < p.hidden; c += blockDim.x * zero.N) zero.template store<STREAM>(p.out, (size_t)r * p.out_stride + c, p.hidden - c);
}

// STREAM, of the kernels below: whether what a pass reads and writes is more than the last-level cache holds. Then the rows written
// (copies, and gradients), or the rows read for a sum, are marked as not used again. One pass leaves the caches to the next, so that
// they are measured together, bf16 rows of 7168 values, 8 slots a token: copies of 16384 tokens and their sum 817 us (5.2 TB/s, what
// a large copy reaches) against 846, a sum of 8191 and its gradient 599 against 624; marked loads alone 841 and 610, stores alone
// 828 and 620. Rows that fit are not marked (3001 tokens of 5120 values, 6 slots: copies 35 against 39, sums 34 against 41).

// A wave takes 64 pieces of a token's row, and writes them topk times.
template <int DT, bool STREAM>
__global__ __launch_bounds__(64 * TOK_WAVES) void sort_tokens_kernel(TokenParams p)
{
    const int t = blockIdx.x, c = (tok_unit() * 64 + (threadIdx.x & 63)) * TokPiece<DT>::N;
    if (t >= p.rows) return tok_zero_tail<DT, STREAM>(p);
    if (c >= p.hidden) return;
    TokPiece<DT> x;
    x.load(p.in, (size_t)t * p.in_stride + c, p.hidden - c);
    for (int k = 0; k < p.topk; ++k) {
        const int at = p.position[(size_t)t * p.topk + k];
        if (at >= 0 && at < p.sorted_rows) x.template store<STREAM>(p.out, (size_t)at * p.out_stride + c, p.hidden - c);
    }
}

// A wave takes 64 pieces of a token's sum, all of its rows' at once. fp32 sums in the order of the slots, rounded once.
template <int DT, bool STREAM>
__global__ __launch_bounds__(64 * (STREAM ? TOK_SUM_WAVES : TOK_WAVES)) void combine_tokens_kernel(TokenParams p)
{
    constexpr int N = TokPiece<DT>::N;
    const int t = blockIdx.x, c = (tok_unit() * 64 + (threadIdx.x & 63)) * N;
    if (c >= p.hidden) return;
    float sum[N] = {};
    for (int k0 = 0; k0 < p.topk; k0 += 8) {
        TokPiece<DT> y[8];
        float w[8];
        bool here[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const size_t slot = (size_t)t * p.topk + k0 + k;
            const int at = k0 + k < p.topk ? p.position[slot] : -1;
            here[k] = at >= 0 && at < p.sorted_rows;
            w[k] = here[k] && p.weights ? p.weights[slot] : 1.0f;
            if (here[k]) y[k].template load<STREAM>(p.in, (size_t)at * p.in_stride + c, p.hidden - c);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (here[k])
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = __builtin_fmaf(w[k], y[k].get(i), sum[i]);
    }
    TokPiece<DT> out, r;
    r.v = 0;
    if (p.residual) r.load(p.residual, (size_t)t * p.residual_stride + c, p.hidden - c);
#pragma unroll
    for (int i = 0; i < N; ++i) out.set(i, p.residual ? sum[i] + r.get(i) : sum[i]);
    out.store(p.out, (size_t)t * p.out_stride + c, p.hidden - c);
}

// A wave takes a slot: its row's gradient, and its weight's, a sum over the row that no other wave shares (8191 x 8 rows of 7168: 2 GB in
// 425 us, 4.8 TB/s).
template <int DT, bool STREAM>
__global__ __launch_bounds__(64 * TOK_WAVES) void combine_grad_kernel(TokenParams p)
{
    constexpr int N = TokPiece<DT>::N;
    const int t = blockIdx.x, k = tok_unit(), lane = threadIdx.x & 63;
    if (t >= p.rows) return tok_zero_tail<DT, STREAM>(p);
    if (k >= p.topk) return;
    const size_t slot = (size_t)t * p.topk + k;
    const int at = p.position[slot];
    float dot = 0;
    if (at >= 0 && at < p.sorted_rows) {
        const float w = p.weights[slot];
#pragma unroll 4
        for (int c = lane * N; c < p.hidden; c += 64 * N) {
            TokPiece<DT> g, y, d;
            g.load(p.in, (size_t)t * p.in_stride + c, p.hidden - c);
            y.load(p.y, (size_t)at * p.y_stride + c, p.hidden - c);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dot = __builtin_fmaf(g.get(i), y.get(i), dot);
                d.set(i, w * g.get(i));
            }
            d.template store<STREAM>(p.out, (size_t)at * p.out_stride + c, p.hidden - c);
        }
        for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
    }
    if (lane == 0) p.grad_weights[slot] = dot;
}

// Launches of at most so many tokens, whose threads stay below 2^32. (A loop over tokens in the kernels costs the scalar loads of the
// positions, which the stores before them might have changed: 3001 tokens of 5120 values, 6 slots, are summed in 28 us instead of 18.)
constexpr int TOK_LAUNCH = 1 << 21;
constexpr int64_t TOK_CACHE = 256 << 20;
static size_t tok_bytes(int dtype) { return dtype == EVAMX_DTYPE_F32 ? 4 : 2; }

// f(p of the tokens of each launch, whether it is the last) for `rows` tokens; in, residual and out are tokens' rows where `sums`,
// in alone where not.
template <class F>
static void tok_launches(TokenParams p, int dtype, bool sums, F f)
{
    const int rows = p.rows;
    for (int t = 0;; t += TOK_LAUNCH) {
        const bool last = rows - t <= TOK_LAUNCH;
        p.rows = last ? rows - t : TOK_LAUNCH;
        f(p, last);
        if (last) return;
        const size_t n = TOK_LAUNCH, size = tok_bytes(dtype);
        p.position += n * p.topk;
        if (p.weights) p.weights += n * p.topk;
        if (p.grad_weights) p.grad_weights += n * p.topk;
        if (p.residual) p.residual = (const char*)p.residual + n * p.residual_stride * size;
        if (sums) p.out = (char*)p.out + n * p.out_stride * size;
        else p.in = (const char*)p.in + n * p.in_stride * size;
    }
}

// Workgroups that clear the tail: enough to write at the memory's rate where there is one.
static int tok_tail_groups(int64_t sorted_rows) { return (int)(sorted_rows < 1024 ? sorted_rows : 1024); }

// f(the type, whether a pass of so many values streams)
template <class F>
static void tok_dispatch(int dtype, int64_t values, F f)
{
    auto as = [&](auto dt) {
        if (values * (int64_t)tok_bytes(dtype) > TOK_CACHE) f(dt, std::true_type());
        else f(dt, std::false_type());
    };
    if (dtype == EVAMX_DTYPE_F32) as(std::integral_constant<int, EVAMX_DTYPE_F32>());
    else if (dtype == EVAMX_DTYPE_BF16) as(std::integral_constant<int, EVAMX_DTYPE_BF16>());
    else as(std::integral_constant<int, EVAMX_DTYPE_F16>());
}

static bool tok_sizes_ok(const char* who, int rows, int topk, int n_local)
{
    if (rows < 0 || topk < 1 || topk > TOK_MAX_TOPK || (int64_t)rows * topk > TOK_MAX_SLOTS) {
        set_error("%s: %d rows of %d experts (topk 1..%d, up to 2^26 slots)", who, rows, topk, TOK_MAX_TOPK);
        return false;
    }
    if (n_local < 1 || n_local > TOK_MAX_EXPERTS) {
        set_error("%s: %d experts outside 1..%d", who, n_local, TOK_MAX_EXPERTS);
        return false;
    }
    return true;
}

static bool tok_row_args_ok(const char* who, int dtype, int hidden, int64_t a, int64_t b)
{
    if (dtype != EVAMX_DTYPE_F16 && dtype != EVAMX_DTYPE_BF16 && dtype != EVAMX_DTYPE_F32) { set_error("%s: dtype %d", who, dtype); return false; }
    if (hidden < 1 || hidden > EVAMX_W4_MAX_DIM) { set_error("%s: hidden %d outside 1..%d", who, hidden, EVAMX_W4_MAX_DIM); return false; }
    if (a < hidden || b < hidden) { set_error("%s: strides below the row length", who); return false; }
    return true;
}

static int ord_chunks(int64_t slots, int* chunk)
{
    // 2048 slots a workgroup, 128 a wave, as long as that makes no more chunks than a workgroup can sum up quickly
    int64_t c = (slots + ORD_MAX_CHUNKS - 1) / ORD_MAX_CHUNKS;
    c = c < 2048 ? 2048 : (c + ORD_THREADS - 1) / ORD_THREADS * ORD_THREADS;
    if (chunk) *chunk = (int)c;
    return (int)((slots + c - 1) / c);
}

static TokenParams tok_params(int rows, int hidden, int topk, const int32_t* position, int64_t sorted_rows)
{
    TokenParams p = {};
    p.rows = rows; p.hidden = hidden; p.topk = topk;
    p.position = position; p.sorted_rows = sorted_rows;
    return p;
}

// The parts of 64 pieces in a row.
static int tok_parts(int dtype, int hidden)
{
    const int per = 64 * (dtype == EVAMX_DTYPE_F32 ? 4 : 8);
    return (hidden + per - 1) / per;
}

}  // namespace evamx

using namespace evamx;

extern "C" size_t evamx_expert_order_workspace_bytes(int rows, int topk, int n_local)
{
    set_error("%s", "");
    if (!tok_sizes_ok("evamx_expert_order_workspace_bytes", rows, topk, n_local)) return 0;
    const int chunks = ord_chunks((int64_t)rows * topk, nullptr);
    return chunks <= 1 ? 0 : (size_t)chunks * n_local * sizeof(int32_t);
}

extern "C" int evamx_expert_order(const int64_t* sel, int rows, int topk, int64_t first_expert, int n_local, int32_t* starts,
                                  int32_t* position, void* workspace, size_t workspace_bytes, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!tok_sizes_ok("evamx_expert_order", rows, topk, n_local)) return EVAMX_EINVAL;
    const size_t need = evamx_expert_order_workspace_bytes(rows, topk, n_local);
    if (!starts || (rows && (!sel || !position)) || (need && !workspace)) { set_error("evamx_expert_order: null pointer"); return EVAMX_EINVAL; }
    if (workspace_bytes < need) { set_error("evamx_expert_order: workspace %zu bytes < %zu", workspace_bytes, need); return EVAMX_ENOSPACE; }
    if ((uintptr_t)workspace & 3) { set_error("evamx_expert_order: the workspace must be 4-byte aligned"); return EVAMX_EINVAL; }
    OrderParams p;
    p.sel = sel; p.first = first_expert; p.slots = rows * topk; p.n_local = n_local;
    p.chunks = ord_chunks(p.slots, &p.chunk);
    p.segment = p.chunk / ORD_WAVES;
    p.starts = starts; p.position = position; p.counts = (int32_t*)workspace;
    int bits = 0;
    while ((n_local - 1) >> bits) ++bits;
    const hipStream_t s = (hipStream_t)stream;
    const size_t lds = (size_t)ORD_WAVES * n_local * sizeof(int);
    if (p.chunks <= 1) {
        // one launch; only as long a segment as the slots need (64 at a time)
        p.segment = ((p.slots + ORD_WAVES - 1) / ORD_WAVES + 63) / 64 * 64;
        order_place_kernel<true><<<1, ORD_THREADS, lds, s>>>(p, bits);
    } else {
        order_count_kernel<<<p.chunks, ORD_THREADS, 0, s>>>(p);
        order_place_kernel<false><<<p.chunks, ORD_THREADS, lds, s>>>(p, bits);
    }
    return launched("expert_order");
}

extern "C" int evamx_sort_tokens(const void* x, int dtype, int64_t x_stride, int rows, int hidden, int topk, const int32_t* position,
                                 const int32_t* starts, int n_local, void* out, int64_t out_stride, int64_t out_rows, evamx_stream_t stream)
{
    set_error("%s", "");
    if (out_rows < 0) { set_error("evamx_sort_tokens: %lld sorted rows", (long long)out_rows); return EVAMX_EINVAL; }
    if (!tok_sizes_ok("evamx_sort_tokens", rows, topk, n_local) || !tok_row_args_ok("evamx_sort_tokens", dtype, hidden, x_stride, out_stride))
        return EVAMX_EINVAL;
    if (out_rows == 0) return EVAMX_OK;
    if ((rows && (!x || !position)) || !starts || !out) { set_error("evamx_sort_tokens: null pointer"); return EVAMX_EINVAL; }
    TokenParams p = tok_params(rows, hidden, topk, position, out_rows);
    p.starts = starts; p.n_local = n_local;
    p.in = x; p.in_stride = (size_t)x_stride; p.out = out; p.out_stride = (size_t)out_stride;
    const TokGrid g(tok_parts(dtype, hidden), TOK_WAVES);
    tok_dispatch(dtype, (out_rows + rows) * hidden, [&](auto dt, auto stream_out) {
        tok_launches(p, dtype, false, [&](const TokenParams& q, bool last) {
            sort_tokens_kernel<decltype(dt)::value, decltype(stream_out)::value>
                <<<dim3(q.rows + (last ? tok_tail_groups(out_rows) : 0), g.groups), 64 * g.waves, 0, (hipStream_t)stream>>>(q);
        });
    });
    return launched("sort_tokens");
}

extern "C" int evamx_combine_tokens(const void* y, int dtype, int64_t y_stride, int64_t y_rows, int rows, int hidden, int topk,
                                    const int32_t* position, const float* weights, const void* residual, int64_t residual_stride,
                                    void* out, int64_t out_stride, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!tok_sizes_ok("evamx_combine_tokens", rows, topk, 1) || !tok_row_args_ok("evamx_combine_tokens", dtype, hidden, y_stride, out_stride))
        return EVAMX_EINVAL;
    if (y_rows < 0) { set_error("evamx_combine_tokens: %lld sorted rows", (long long)y_rows); return EVAMX_EINVAL; }
    if (residual && residual_stride < hidden) { set_error("evamx_combine_tokens: strides below the row length"); return EVAMX_EINVAL; }
    if (rows == 0) return EVAMX_OK;
    if ((y_rows && !y) || !position || !out) { set_error("evamx_combine_tokens: null pointer"); return EVAMX_EINVAL; }
    TokenParams p = tok_params(rows, hidden, topk, position, y_rows);
    p.in = y; p.in_stride = (size_t)y_stride; p.weights = weights; p.residual = residual; p.residual_stride = (size_t)residual_stride;
    p.out = out; p.out_stride = (size_t)out_stride;
    tok_dispatch(dtype, ((int64_t)rows * topk + rows) * hidden, [&](auto dt, auto stream_in) {
        constexpr bool STREAM = decltype(stream_in)::value;
        const TokGrid g(tok_parts(dtype, hidden), STREAM ? TOK_SUM_WAVES : TOK_WAVES);
        tok_launches(p, dtype, true, [&](const TokenParams& q, bool) {
            combine_tokens_kernel<decltype(dt)::value, STREAM>
                <<<dim3(q.rows, g.groups), 64 * g.waves, 0, (hipStream_t)stream>>>(q);
        });
    });
    return launched("combine_tokens");
}

extern "C" int evamx_combine_tokens_grad(const void* grad, int dtype, int64_t grad_stride, const void* y, int64_t y_stride, int64_t y_rows,
                                         int rows, int hidden, int topk, const int32_t* position, const int32_t* starts, int n_local,
                                         const float* weights, void* grad_y, int64_t grad_y_stride, float* grad_weights, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!tok_sizes_ok("evamx_combine_tokens_grad", rows, topk, n_local) ||
        !tok_row_args_ok("evamx_combine_tokens_grad", dtype, hidden, grad_stride, grad_y_stride))
        return EVAMX_EINVAL;
    if (y_rows < 0) { set_error("evamx_combine_tokens_grad: %lld sorted rows", (long long)y_rows); return EVAMX_EINVAL; }
    if (y_stride < hidden) { set_error("evamx_combine_tokens_grad: strides below the row length"); return EVAMX_EINVAL; }
    if (!starts || (y_rows && (!y || !grad_y)) || (rows && (!grad || !position || !weights || !grad_weights))) {
        set_error("evamx_combine_tokens_grad: null pointer");
        return EVAMX_EINVAL;
    }
    if (rows == 0 && y_rows == 0) return EVAMX_OK;
    TokenParams p = tok_params(rows, hidden, topk, position, y_rows);
    p.starts = starts; p.n_local = n_local;
    p.in = grad; p.in_stride = (size_t)grad_stride; p.y = y; p.y_stride = (size_t)y_stride; p.weights = weights;
    p.out = grad_y; p.out_stride = (size_t)grad_y_stride; p.grad_weights = grad_weights;
    const TokGrid g(topk, TOK_WAVES);
    tok_dispatch(dtype, (2 * y_rows + rows) * hidden, [&](auto dt, auto stream_out) {
        tok_launches(p, dtype, false, [&](const TokenParams& q, bool last) {
            combine_grad_kernel<decltype(dt)::value, decltype(stream_out)::value>
                <<<dim3(q.rows + (last ? tok_tail_groups(y_rows) : 0), g.groups), 64 * g.waves, 0, (hipStream_t)stream>>>(q);
        });
    });
    return launched("combine_tokens_grad");
}
