// The gradients of act(x W^T + b): D = act'(pre) grad, W's D^T x, the bias's column sums of D. x's, D W, is a product as the
// forward one (tiles.hip).
#include "grads.hpp"

namespace evamx_dense {

// D of eight values of a row. It is rounded to 16 bits, as the matrix cores take it. Bound by memory: 2000 rows of 5120 values, 82 MB
// that the last-level cache still holds, 15 us.
template <class T, bool GATED>
__global__ __launch_bounds__(256) void act_grad_kernel(ActGradParams p)
{
    constexpr bool BF = std::is_same<T, Bf16>::value;
    const int cols = GATED ? p.n_out / 2 : p.n_out, per = (cols + 7) / 8;
    // rows of the experts alone, whose number the host does not know: each workgroup goes on to the next 2048 values
    const int64_t all = (int64_t)p.g.end() * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / per;
        const int n = (int)(at - row * per) * 8, have = cols - n;
        float gr[8], v[8], u[8], dv[8], du[8];
        load8(gr, p.grad + (size_t)row * p.grad_stride + n, have, BF);
        const float* pre = p.pre + (size_t)row * p.n_out + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = u[i] = 0;
        add_floats(v, pre, have);
        if (GATED) add_floats(u, pre + cols, have);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (GATED) {
                const float sg = sigmoid(v[i]), a = v[i] * sg, s = sg * (1.0f + v[i] * (1.0f - sg));
                const bool cut = p.limit > 0, whole_a = !cut || !(a > p.limit), whole_u = !cut || !(fabsf(u[i]) > p.limit);
                dv[i] = whole_a ? gr[i] * (cut ? within(u[i], p.limit) : u[i]) * s : 0.0f;
                du[i] = whole_u ? gr[i] * (cut ? at_most(a, p.limit) : a) : 0.0f;
            } else {
                dv[i] = gr[i] * slope(v[i], p.act);
            }
        }
        uint16_t* out = p.out + (size_t)row * p.out_stride + n;
        auto store = [&](uint16_t* to, const float (&d)[8]) {
            if (have >= 8) {
                u16x8 o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = T::put(d[i]);
                *(u16x8_loose*)to = o;
            } else {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < have) to[i] = T::put(d[i]);
            }
        };
        store(out, dv);
        if (GATED) store(out + cols, du);
        if (have <= 8) {                                                    // the row's end: zeros up to the stride
            for (int i = p.n_out; i < (int)p.out_stride; ++i) p.out[(size_t)row * p.out_stride + i] = 0;
        }
    }
}

// Tiles of n that a run of tiles takes together for all of k: eight share more of what they read; with the experts' shorter sums,
// whose results are most of the traffic, one, so that rows are written whole (32 experts of about 128 rows, 4096 by 7168: 655 us
// against 700; one of 8192 rows: 411 against 389).
__device__ __forceinline__ int deep_of(const WeightGradParams& p) { return p.g.starts ? 1 : 8; }

// W's gradient: result rows q = n of W, p = k. The sum runs over the expert's rows, in tiles of 64. A workgroup takes one tile after
// another: the next one's first k-tiles are asked for before this one's results are stored, so that with few rows an expert, where
// the stores are most of the work, they need not be waited for.
template <class T, int WP, int WQ, int QB>
__global__ __launch_bounds__(64 * WP * WQ, 2) void weight_grad_kernel(WeightGradParams p, int tiles)
{
    constexpr int PB = 4;
    typedef Gemm<T, true, true, WP, WQ, PB, QB, 1, 2> G;
    __shared__ __attribute__((aligned(1024))) char lds[G::STAGES_BYTES];
    const int pt = (p.n_in + G::TP - 1) / G::TP, qt = (p.n_out + G::TQ - 1) / G::TQ, splits = p.plan.splits;
    typename G::P a;
    typename G::Q b;
    int e, p0, q0, k0, k1, split;
    // work item u: tile by tile of an expert (and split), each XCD a contiguous run of them, deep_of tiles of n by all of k at a time
    auto take = [&](int u) {
        const int per = (tiles + 7) / 8, unit = u / (8 * per), in = u - unit * 8 * per, at = (in & 7) * per + in / 8;
        if (at >= tiles) return false;
        split = unit % splits;
        e = unit / splits;
        const int most = deep_of(p), band = at / (most * pt), in_band = at - band * most * pt, deep = qt - most * band < most ? qt - most * band : most;
        q0 = G::TQ * (most * band + in_band % deep);
        p0 = G::TP * (in_band / deep);
        const int begin = p.g.starts ? p.g.start(e) : 0, end = p.g.starts ? p.g.start(e + 1) : p.g.rows, count = end > begin ? end - begin : 0;
        a.init(p.x + (size_t)begin * p.x_stride + p0, p.x_stride, count, p.x_cols - p0, [](int n) { return n; });
        b.init(p.d + (size_t)begin * p.d_stride + q0, p.d_stride, count, p.d_cols - q0, [](int n) { return n; });
        const int kt = (count + TILE_K - 1) / TILE_K;
        k0 = splits > 1 ? (int)((long)kt * split / splits) : 0;
        k1 = splits > 1 ? (int)((long)kt * (split + 1) / splits) : kt;
        return true;
    };
    const int units = 8 * ((tiles + 7) / 8) * p.g.experts * splits, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    while (u < units && !take(u)) u += gridDim.x;
    if (u >= units) return;
    G::begin(a, b, lds, k0, k1);
    bool stored = false;                                               // 2 QB stores of the last tile's results are under way
    for (;;) {
        f32x4 acc[PB][QB] = {};
        const size_t row0 = splits > 1 ? (size_t)split * p.n_out : (size_t)e * p.n_out;
        const int to_p = p0 + 64 * G::wp(), to_q = q0 + 16 * QB * G::wq();
        const bool whole = p0 + G::TP <= p.n_in && q0 + G::TQ <= p.n_out && splits == 1;
        G::template run<2 * QB>(acc, a, b, lds, k0, k1, stored);
        stored = whole;
        do u += gridDim.x;
        while (u < units && !take(u));
        if (u < units) G::begin(a, b, lds, k0, k1);
        if (whole) {
            uint16_t* at = p.out + (row0 + to_q + (c & 7)) * p.n_in + to_p + 32 * (c >> 3) + 16 * (g & 1) + 8 * (g >> 1);
            auto all = [&](auto stream) {
#pragma unroll
                for (int j = 0; j < QB; ++j) {
                    const f32x4 sums[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
                    u16x8 v[2];
                    lined<T>(sums, v);
#pragma unroll
                    for (int i = 0; i < 2; ++i) store16<decltype(stream)::value>(at + (size_t)(2 * j + i) * 8 * p.n_in, v[i]);
                }
            };
            if (p.stream) all(std::true_type());
            else all(std::false_type());
        } else {
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                const int q = to_q + 16 * j + c;
                if (q >= p.n_out) continue;
#pragma unroll
                for (int i = 0; i < PB; ++i) {
                    const int k = to_p + 16 * i + 4 * g;
                    const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                    if (splits > 1) {
                        store_floats(p.part + (row0 + q) * p.n_in + k, v, p.n_in - k);
                    } else {
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            if (k + h < p.n_in) p.out[(row0 + q) * p.n_in + k + h] = T::put(v[h]);
                    }
                }
            }
        }
        if (u >= units) return;
    }
}

// Rows of n values at any address to rows of whole 16 bytes, zeros behind the last value, for the tiles: eight values a lane, as whole
// words and a shift where the row goes on at both ends (2000 x 1001 by 999 x 1001: 34 us with both copies, 62 with such loads in the
// tiles).
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t* from, size_t stride, size_t matrix_stride, int rows, int64_t all, int n, uint16_t* to)
{
    const int per = (n + 7) / 8;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all * per; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / per;
        const int v = (int)(at - row * per) * 8;
        const uint16_t* p = from + (size_t)(row / rows) * matrix_stride + (size_t)(row % rows) * stride + v;
        u16x8 x = (u16x8)(uint16_t)0;
        if (v > 0 && v + 10 <= n) {
            x = load8_shifted(p);
        } else if (v + 8 <= n) {
            x = *(const u16x8_loose*)p;
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (v + i < n) x[i] = p[i];
        }
        *(u16x8*)(to + (size_t)row * (8 * per) + v) = x;
    }
}

int launch_pad(const uint16_t* from, size_t stride, size_t matrix_stride, int rows, int count, int n, uint16_t* to, hipStream_t s)
{
    const int64_t all = (int64_t)rows * count;
    const int64_t groups = (all * ((n + 7) / 8) + 255) / 256;
    pad_kernel<<<(unsigned)(groups < 1 << 22 ? groups : 1 << 22), 256, 0, s>>>(from, stride, matrix_stride, rows, all, n, to);
    return launched("linear");
}

// Sums of `count` arrays of n values each, rounded; array s of value i of matrix y: part[(y * count + s) * n + i].
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int count, int64_t n, uint16_t* out)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0;
#pragma unroll 8
    for (int s = 0; s < count; ++s) v += part[((size_t)blockIdx.y * count + s) * n + i];
    out[(size_t)blockIdx.y * n + i] = T::put(v);
}

// Sums of an expert's rows of D over one of `parts` runs of them, eight columns a lane; the waves' sums meet in LDS. 2000 rows of 5120
// values in 26 runs: 6.3 us, and 4.2 for the sum of these.
template <class T>
__global__ __launch_bounds__(256) void column_sums_kernel(ColumnSumParams p)
{
    constexpr bool BF = std::is_same<T, Bf16>::value;
    __shared__ float sums[4][64 * 9];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (blockIdx.x * 64 + lane) * 8, e = blockIdx.y;
    const int begin = p.g.starts ? p.g.start(e) : 0, end = p.g.starts ? p.g.start(e + 1) : p.g.rows, count = end > begin ? end - begin : 0;
    const int r0 = begin + (int)((int64_t)count * blockIdx.z / p.parts), r1 = begin + (int)((int64_t)count * (blockIdx.z + 1) / p.parts);
    float v[8] = {};
    if (n < p.n_out) {
#pragma unroll 4
        for (int r = r0 + wave; r < r1; r += 4) {
            float d[8];
            load8(d, p.d + (size_t)r * p.d_stride + n, p.n_out - n, BF);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += d[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[wave][lane * 9 + i] = v[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int col = blockIdx.x * 512 + i, at = (i >> 3) * 9 + (i & 7);
        if (col >= p.n_out) continue;
        const float s = (sums[0][at] + sums[1][at]) + (sums[2][at] + sums[3][at]);
        if (p.parts > 1) p.part[((size_t)e * p.parts + blockIdx.z) * p.n_out + col] = s;
        else p.out[(size_t)e * p.n_out + col] = T::put(s);
    }
}

template <class F>
static void by_type(int dtype, F f)
{
    if (dtype == EVAMX_DTYPE_BF16) f(Bf16());
    else f(F16());
}

int launch_act_grad(const ActGradParams& p, int dtype, hipStream_t s)
{
    const int cols = p.act == EVAMX_ACT_SWIGLU ? p.n_out / 2 : p.n_out;
    const int64_t most = ceil_div((int64_t)p.g.rows * ceil_div(cols, 8), 256);
    const unsigned grid = (unsigned)(most < 16 * CUS ? most : 16 * CUS);
    by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        if (p.act == EVAMX_ACT_SWIGLU) act_grad_kernel<T, true><<<grid, 256, 0, s>>>(p);
        else act_grad_kernel<T, false><<<grid, 256, 0, s>>>(p);
    });
    return launched("linear_grad");
}

template <class T, int WP, int WQ, int QB>
static void launch_weight_grad_as(const WeightGradParams& p, hipStream_t s)
{
    const int64_t tiles = (int64_t)ceil_div(p.n_in, 64 * WP) * ceil_div(p.n_out, 16 * QB * WQ);
    const int64_t units = 8 * ceil_div(tiles, 8) * (int64_t)p.g.experts * p.plan.splits, at_once = WP * WQ == 8 ? CUS : 2 * CUS;
    weight_grad_kernel<T, WP, WQ, QB><<<(unsigned)(units < at_once ? units : at_once), 64 * WP * WQ, 0, s>>>(p, (int)tiles);
}

int launch_weight_grad(const WeightGradParams& p, int dtype, hipStream_t s)
{
    by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        if (p.plan.size == TILES_256) launch_weight_grad_as<T, 4, 2, 8>(p, s);
        else launch_weight_grad_as<T, 2, 2, 4>(p, s);
        if (p.plan.splits > 1) {
            const int64_t n = (int64_t)p.n_out * p.n_in;
            sum_parts_kernel<T><<<dim3((unsigned)ceil_div(n, 256), 1), 256, 0, s>>>(p.part, p.plan.splits, n, p.out);
        }
    });
    return launched("linear_grad");
}

int launch_column_sums(const ColumnSumParams& p, int dtype, hipStream_t s)
{
    by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        column_sums_kernel<T><<<dim3(ceil_div(p.n_out, 512), p.g.experts, p.parts), 256, 0, s>>>(p);
        if (p.parts > 1) sum_parts_kernel<T><<<dim3(ceil_div(p.n_out, 256), p.g.experts), 256, 0, s>>>(p.part, p.parts, p.n_out, p.out);
    });
    return launched("linear_grad");
}

}  // namespace evamx_dense
