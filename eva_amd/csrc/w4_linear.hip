// y = x W^T (+ bias) on 4-bit weights with group scales (w4.hpp).
#include "evamx_internal.hpp"
#include "w4.hpp"

namespace evamx {

__device__ __forceinline__ float w4_bias(const void* b, int n, int bf16)
{
    return bf16 ? __builtin_bit_cast(float, (uint32_t)((const uint16_t*)b)[n] << 16) : (float)((const w4_half*)b)[n];
}

// One workgroup 16 columns by 16 rows, its four waves every fourth quad of k-tiles.
template <int SG, bool ZERO>
__global__ __launch_bounds__(256) void w4_linear_kernel(const w4_half* __restrict__ x, const float* __restrict__ row_scale, int rows,
                                                        W4Mat m, const void* __restrict__ bias, void* __restrict__ y, size_t y_stride,
                                                        int bf16)
{
    __shared__ w4_f32x4 part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nt = blockIdx.x, r0 = 16 * blockIdx.y, row = r0 + (lane & 15);
    w4_f32x4 acc = {0, 0, 0, 0};
    w4_accumulate<SG, ZERO>(acc, m, 0, nt, row < rows ? x + (size_t)row * m.kt * W4_TILE_K + 8 * (lane >> 4) : nullptr, wave, 4);
    part[wave][lane] = acc;
    __syncthreads();
    const int r = 4 * (lane >> 4) + wave, n = 16 * nt + (lane & 15);      // wave w joins and stores rows 4 g + w
    if (r0 + r >= rows || n >= m.n_out) return;
    float v = 0;
    for (int w = 0; w < 4; ++w) v += part[w][lane][wave];
    v *= row_scale[r0 + r];
    if (bias) v += w4_bias(bias, n, bf16);
    w4_store(y, (size_t)(r0 + r) * y_stride + n, v, bf16);
}

}  // namespace evamx

using namespace evamx;

extern "C" size_t evamx_w4_linear_workspace_bytes(int rows, int n_in)
{
    if (rows < 1 || rows > 65536 || n_in < 1 || n_in > EVAMX_W4_MAX_DIM) return 0;
    return w4_align((size_t)rows * 4) + w4_align((size_t)rows * w4_ceil(n_in, W4_TILE_K) * W4_TILE_K * 2);
}

extern "C" int evamx_w4_linear(const void* x, int x_dtype, int64_t x_stride, int rows, const evamx_w4_weight* w, const void* bias,
                               void* y, int64_t y_stride, void* workspace, size_t workspace_bytes, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!w4_weight_ok(w, "evamx_w4_linear")) return EVAMX_EINVAL;
    if (!x || !y || !workspace) { set_error("evamx_w4_linear: null pointer"); return EVAMX_EINVAL; }
    if (w->count != 1) { set_error("evamx_w4_linear: a stack of %d matrices", w->count); return EVAMX_EINVAL; }
    if (x_dtype != EVAMX_DTYPE_F16 && x_dtype != EVAMX_DTYPE_BF16) { set_error("evamx_w4_linear: x_dtype %d", x_dtype); return EVAMX_EINVAL; }
    if (rows < 1 || rows > 65536) { set_error("evamx_w4_linear: rows %d outside 1..65536", rows); return EVAMX_EINVAL; }
    if (x_stride < w->n_in || y_stride < w->n_out) { set_error("evamx_w4_linear: strides below the row lengths"); return EVAMX_EINVAL; }
    if ((uintptr_t)workspace & 15) { set_error("evamx_w4_linear: the workspace must be 16-byte aligned"); return EVAMX_EINVAL; }
    const size_t need = evamx_w4_linear_workspace_bytes(rows, w->n_in);
    if (workspace_bytes < need) { set_error("evamx_w4_linear: workspace %zu bytes < %zu", workspace_bytes, need); return EVAMX_ENOSPACE; }
    const hipStream_t s = (hipStream_t)stream;
    float* rs = (float*)workspace;
    w4_half* xh = (w4_half*)((char*)workspace + w4_align((size_t)rows * 4));
    const int bf16 = x_dtype == EVAMX_DTYPE_BF16;
    w4_launch_rows(x, x_dtype, (size_t)x_stride, rows, w->n_in, xh, rs, s);
    const W4Mat m = w4_mat(*w);
    const dim3 grid(w4_ceil(m.n_out, W4_TILE_N), w4_ceil(rows, 16));
    w4_dispatch(*w, [&](auto sg, auto zero) {
        w4_linear_kernel<decltype(sg)::value, decltype(zero)::value><<<grid, 256, 0, s>>>(xh, rs, rows, m, bias, y, (size_t)y_stride, bf16);
    });
    return launched("w4_linear");
}
