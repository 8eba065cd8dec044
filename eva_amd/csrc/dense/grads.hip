// The gradients of act(x W^T + b): D = act'(pre) grad, W's D^T x, the bias's column sums of D. x's, D W, is a product as the
// forward one (tiles.hip).
#include <stdlib.h>

#include "grads.hpp"

namespace evamx_dense {

// D of eight values of a row. It is rounded to 16 bits, as the matrix cores take it.
template <class T, bool GATED>
__global__ __launch_bounds__(256) void act_grad_kernel(ActGradParams p)
{
    constexpr bool BF = std::is_same<T, Bf16>::value;
    const int cols = GATED ? p.n_out / 2 : p.n_out, per = (cols + 7) / 8;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = at / per;
    const int n = (int)(at % per) * 8, have = cols - n;
    if (row >= p.g.end()) return;
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
}

// W's gradient: result rows q = n of W, p = k. The sum runs over the expert's rows, in tiles of 64.
template <class T, bool LOOSE, int WP, int WQ, int QB, int KW>
__global__ __launch_bounds__(64 * WP * WQ * KW, 2) void weight_grad_kernel(WeightGradParams p)
{
    constexpr int PB = 4;
    typedef Gemm<T, true, true, WP, WQ, PB, QB, KW, 2, LOOSE> G;
    __shared__ __attribute__((aligned(1024))) char lds[G::LDS];
    const int pt = (p.n_in + G::TP - 1) / G::TP, qt = (p.n_out + G::TQ - 1) / G::TQ, tiles = pt * qt;
    // an XCD takes a contiguous run of tiles, eight tiles of n by all of k at a time
    const int per = (tiles + 7) / 8, at = (blockIdx.x & 7) * per + blockIdx.x / 8;
    if ((int)blockIdx.x / 8 >= per || at >= tiles) return;
    const int band = at / (8 * pt), in_band = at - band * 8 * pt, deep = qt - 8 * band < 8 ? qt - 8 * band : 8;
    const int q0 = G::TQ * (8 * band + in_band % deep), p0 = G::TP * (in_band / deep), e = blockIdx.y;
    const int begin = p.g.starts ? p.g.start(e) : 0, end = p.g.starts ? p.g.start(e + 1) : p.g.rows, count = end > begin ? end - begin : 0;
    typename G::P a;
    typename G::Q b;
    a.init(p.x + (size_t)begin * p.x_stride + p0, p.x_stride, count, p.n_in - p0, [](int n) { return n; });
    b.init(p.d + (size_t)begin * p.d_stride + q0, p.d_stride, count, p.n_out - q0, [](int n) { return n; });
    f32x4 acc[PB][QB] = {};
    const int kt = (count + TILE_K - 1) / TILE_K, k0 = (int)((long)kt * blockIdx.z / p.splits), k1 = (int)((long)kt * (blockIdx.z + 1) / p.splits);
    if (!G::run(acc, a, b, lds, k0, k1)) return;
    const int lane = threadIdx.x & 63, wp = G::wp(), wq = G::wq(), k = p0 + 64 * wp + 8 * (lane & 7), have = p.n_in - k;
    rows_of<PB, QB>(acc, lds, wq * WP + wp, [&](const float* mine, int first, int count) {
        if (have <= 0) return;
        for (int r = lane >> 3; r < count; r += 8) {
            const int q = q0 + 16 * QB * wq + first + r;
            if (q >= p.n_out) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mine[r * OUT_ROW + 8 * (lane & 7) + i];
            if (p.splits > 1) {
                store_floats(p.part + ((size_t)blockIdx.z * p.n_out + q) * p.n_in + k, v, have);
                continue;
            }
            uint16_t* out = p.out + ((size_t)e * p.n_out + q) * p.n_in + k;
            if (have >= 8) {
                u16x8 o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = T::put(v[i]);
                *(u16x8_loose*)out = o;
            } else {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < have) out[i] = T::put(v[i]);
            }
        }
    });
}

// Sums of `count` arrays of n values each, rounded; array s of value i of matrix y: part[(y * count + s) * n + i].
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int count, int64_t n, uint16_t* out)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0;
    for (int s = 0; s < count; ++s) v += part[((size_t)blockIdx.y * count + s) * n + i];
    out[(size_t)blockIdx.y * n + i] = T::put(v);
}

// Sums of an expert's rows of D over one of `parts` runs of them, eight columns a lane; the waves' sums meet in LDS.
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
    const unsigned grid = (unsigned)ceil_div((int64_t)p.g.rows * ceil_div(cols, 8), 256);
    by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        if (p.act == EVAMX_ACT_SWIGLU) act_grad_kernel<T, true><<<grid, 256, 0, s>>>(p);
        else act_grad_kernel<T, false><<<grid, 256, 0, s>>>(p);
    });
    return launched("linear_grad");
}

template <class T, bool LOOSE, int WP, int WQ, int QB, int KW>
static void launch_weight_grad_as(const WeightGradParams& p, hipStream_t s)
{
    const int64_t tiles = (int64_t)ceil_div(p.n_in, 64 * WP) * ceil_div(p.n_out, 16 * QB * WQ);
    weight_grad_kernel<T, LOOSE, WP, WQ, QB, KW><<<dim3((unsigned)(8 * ceil_div(tiles, 8)), p.g.experts, p.splits), 64 * WP * WQ * KW, 0, s>>>(p);
}

int launch_weight_grad(const WeightGradParams& p, int dtype, bool loose, hipStream_t s)
{
    by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        const int64_t big = (int64_t)ceil_div(p.n_in, 256) * ceil_div(p.n_out, 256) * p.g.experts;
        static const char* force = getenv("DW_SIZE");
        const int size = force ? atoi(force) : p.splits == 1 && big >= 200 ? 2 : 0;
        if (loose) launch_weight_grad_as<T, true, 2, 1, 8, 2>(p, s);
        else if (size == 2) launch_weight_grad_as<T, false, 4, 2, 8, 1>(p, s);
        else if (size == 1) launch_weight_grad_as<T, false, 2, 2, 4, 1>(p, s);
        else launch_weight_grad_as<T, false, 2, 1, 8, 2>(p, s);
        if (p.splits > 1) {
            const int64_t n = (int64_t)p.n_out * p.n_in;
            sum_parts_kernel<T><<<dim3((unsigned)ceil_div(n, 256), 1), 256, 0, s>>>(p.part, p.splits, n, p.out);
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
