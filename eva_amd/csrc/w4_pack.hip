// 4-bit weights: the layout the products read (w4.hpp), made once per matrix and read back, and rows of activations made
// ready for them.
#include "evamx_internal.hpp"
#include "w4.hpp"

namespace evamx {

// One thread a dword of the packed codes: 8 nibbles of row n at k = 128 t + 32 j + 8 g, read at once where rows are whole dwords.
// Done once per stack, when it is loaded (257 experts of 7168 x 2048, 5.8 GB of codes: about 4 ms).
template <bool DWORDS>
__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const uint8_t* __restrict__ src, W4Mat m, uint32_t* __restrict__ dst, size_t total)
{
    const size_t row_bytes = (size_t)(m.n_in + 1) / 2;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t tile = i / W4_TILE_DWORDS;
        const int r = (int)(i % W4_TILE_DWORDS), lane = r >> 2, j = r & 3;
        const size_t mat = tile / m.tiles, in_mat = tile % m.tiles;
        const size_t n = in_mat / m.kt * W4_TILE_N + (lane & 15);
        const int k = (int)(in_mat % m.kt) * W4_TILE_K + 32 * j + 8 * (lane >> 4);
        uint32_t out = 0;
        if (n < (size_t)m.n_out) {
            const uint8_t* row = src + (mat * m.n_out + n) * row_bytes;
            if constexpr (DWORDS) {
                if (k < m.n_in) {
                    const uint32_t d = *(const uint32_t*)(row + (k >> 1)), lo = d & 0x0f0f0f0fu, hi = (d >> 4) & 0x0f0f0f0fu;
                    const uint32_t a = lo | lo >> 4, b = hi | hi >> 4;            // bytes 0 and 2 hold two nibbles each
                    out = (a & 0xffu) | (a >> 8 & 0xff00u) | (b & 0xffu) << 16 | (b & 0xff0000u) << 8;
                }
            } else
#pragma unroll
            for (int p = 0; p < 4; ++p) {                        // a byte holds k + 2 p (low) and k + 2 p + 1 (high)
                if (k + 2 * p >= m.n_in) break;
                uint32_t b = row[(k >> 1) + p];
                if (k + 2 * p + 1 >= m.n_in) b &= 15;
                out |= (b & 15) << (4 * p) | (b >> 4) << (4 * p + 16);
            }
        }
        dst[i] = out;
    }
}

// One thread a group of the packed scales and zero points; a source group spans src_group / (128 / SG) of them.
__global__ __launch_bounds__(256) void w4_pack_groups_kernel(const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                             int src_group, W4Mat m, int sg, uint16_t* __restrict__ out_s,
                                                             uint8_t* __restrict__ out_z, size_t total)
{
    const int group = W4_TILE_K / sg, src_n = (m.n_in + src_group - 1) / src_group;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t mat = i / m.groups, r = i % m.groups;
        const int g = (int)(r % sg), col = (int)(r / sg % W4_TILE_N);
        const size_t tile = r / (sg * W4_TILE_N);
        const size_t n = tile / m.kt * W4_TILE_N + col;
        const int k = (int)(tile % m.kt) * W4_TILE_K + g * group;
        const bool in = n < (size_t)m.n_out && k < m.n_in;
        const size_t at = in ? (mat * m.n_out + n) * src_n + k / src_group : 0;
        out_s[i] = in ? scales[at] : 0;
        if (zeros) out_z[i] = in ? zeros[at] : 0;
    }
}

// W in fp32, one thread a value: scale * (code - zero), both exact before the one rounding of the product.
__global__ __launch_bounds__(256) void w4_dequant_kernel(W4Mat m, int sg, float* __restrict__ out, size_t total)
{
    const size_t mat_size = (size_t)m.n_out * m.n_in;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t mat = i / mat_size, r = i % mat_size;
        const size_t n = r / m.n_in;
        const int k = (int)(r % m.n_in), nt = (int)(n / W4_TILE_N), col = (int)(n % W4_TILE_N);
        const int kt = k / W4_TILE_K, in_tile = k % W4_TILE_K;
        const int j = in_tile / 32, g = in_tile / 8 % 4, e = in_tile % 8;
        const size_t tile = (size_t)nt * m.kt + kt;
        const uint32_t w = m.codes[(mat * m.tiles + tile) * W4_TILE_DWORDS + (col + 16 * g) * 4 + j];
        const int q = (w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15;
        const size_t at = mat * m.groups + (tile * W4_TILE_N + col) * sg + in_tile * sg / W4_TILE_K;
        out[i] = w4_scale(m.scales[at], m.bf16) * (float)(q - (m.zeros ? (int)(m.zeros[at] & W4_ZERO_MAX) : 8));
    }
}

// One workgroup a row.
template <int SRC>
__global__ __launch_bounds__(256) void w4_rows_kernel(const char* __restrict__ src, size_t stride, bool aligned, int n_in, int n_pad,
                                                      w4_half* __restrict__ dst, float* __restrict__ scale)
{
    __shared__ uint32_t part[4];
    W4ReadyRow<SRC, 256, false> row{src + blockIdx.x * stride, n_in, n_pad, aligned, (int)threadIdx.x};
    row.load();
    const float f = row.finish(dst + blockIdx.x * (size_t)n_pad, 0, part);
    if (threadIdx.x == 0) scale[blockIdx.x] = f;
}

void w4_launch_rows(const void* src, int src_dtype, size_t src_stride, int rows, int n_in, void* dst, float* scale, hipStream_t stream)
{
    const int n_pad = w4_ceil(n_in, W4_TILE_K) * W4_TILE_K;
    const bool aligned = (((uintptr_t)src | (2 * src_stride)) & 15) == 0;
    if (src_dtype == EVAMX_DTYPE_F16)
        w4_rows_kernel<EVAMX_DTYPE_F16><<<rows, 256, 0, stream>>>((const char*)src, src_stride * 2, aligned, n_in, n_pad, (w4_half*)dst, scale);
    else
        w4_rows_kernel<EVAMX_DTYPE_BF16><<<rows, 256, 0, stream>>>((const char*)src, src_stride * 2, aligned, n_in, n_pad, (w4_half*)dst, scale);
}

static int w4_grid(size_t total)
{
    const size_t b = (total + 255) / 256;
    return (int)(b < 65536 ? b : 65536);
}

// The group sizes the kernels are built for; others are stored as the largest of these that divides them.
static bool w4_stored_group(int g) { return g == 32 || g == 64 || g == 128; }

bool w4_weight_ok(const evamx_w4_weight* w, const char* who)
{
    if (!w || !w->codes || !w->scales) { set_error("%s: null weight", who); return false; }
    if (w->count < 1 || w->count > 1024 || w->n_out < 1 || w->n_out > EVAMX_W4_MAX_DIM || w->n_in < 1 || w->n_in > EVAMX_W4_MAX_DIM) {
        set_error("%s: weight of %d matrices [%d, %d] outside 1..1024 and 1..%d", who, w->count, w->n_out, w->n_in, EVAMX_W4_MAX_DIM);
        return false;
    }
    if (!w4_stored_group(w->group)) { set_error("%s: stored group %d not in {32, 64, 128}", who, w->group); return false; }
    if (w->scale_dtype != EVAMX_DTYPE_F16 && w->scale_dtype != EVAMX_DTYPE_BF16) {
        set_error("%s: scale_dtype %d", who, w->scale_dtype);
        return false;
    }
    if (((uintptr_t)w->codes | (uintptr_t)w->scales | (uintptr_t)w->zeros) & 15) {
        set_error("%s: packed weights must be 16-byte aligned", who);
        return false;
    }
    return true;
}

}  // namespace evamx

using namespace evamx;

extern "C" int evamx_w4_stored_group(int group)
{
    if (group < 32 || group % 32) return 0;
    return group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32;
}

extern "C" size_t evamx_w4_code_bytes(int count, int n_out, int n_in)
{
    if (count < 1 || n_out < 1 || n_in < 1 || n_out > EVAMX_W4_MAX_DIM || n_in > EVAMX_W4_MAX_DIM || count > 1024) return 0;
    return (size_t)count * w4_ceil(n_out, W4_TILE_N) * w4_ceil(n_in, W4_TILE_K) * (W4_TILE_DWORDS * 4);
}

extern "C" size_t evamx_w4_group_count(int count, int n_out, int n_in, int group)
{
    if (!w4_stored_group(group) || evamx_w4_code_bytes(count, n_out, n_in) == 0) return 0;
    return (size_t)count * w4_ceil(n_out, W4_TILE_N) * w4_ceil(n_in, W4_TILE_K) * (W4_TILE_N * (W4_TILE_K / group));
}

extern "C" int evamx_w4_pack(const uint8_t* codes, const void* scales, const uint8_t* zeros, int group, const evamx_w4_weight* w,
                             evamx_stream_t stream)
{
    set_error("%s", "");
    if (!w4_weight_ok(w, "evamx_w4_pack")) return EVAMX_EINVAL;
    if (!codes || !scales || (zeros == nullptr) != (w->zeros == nullptr)) {
        set_error("evamx_w4_pack: null pointer, or zero points on one side only");
        return EVAMX_EINVAL;
    }
    if (evamx_w4_stored_group(group) != w->group) {
        set_error("evamx_w4_pack: a group of %d is stored as %d, not %d", group, evamx_w4_stored_group(group), w->group);
        return EVAMX_EINVAL;
    }
    const W4Mat m = w4_mat(*w);
    const size_t dwords = (size_t)w->count * m.tiles * W4_TILE_DWORDS, groups = (size_t)w->count * m.groups;
    if (w->n_in % 8 == 0 && ((uintptr_t)codes & 3) == 0)
        w4_pack_codes_kernel<true><<<w4_grid(dwords), 256, 0, (hipStream_t)stream>>>(codes, m, const_cast<uint32_t*>(m.codes), dwords);
    else
        w4_pack_codes_kernel<false><<<w4_grid(dwords), 256, 0, (hipStream_t)stream>>>(codes, m, const_cast<uint32_t*>(m.codes), dwords);
    w4_pack_groups_kernel<<<w4_grid(groups), 256, 0, (hipStream_t)stream>>>((const uint16_t*)scales, zeros, group, m, W4_TILE_K / w->group,
                                                                        const_cast<uint16_t*>(m.scales),
                                                                        const_cast<uint8_t*>(m.zeros), groups);
    return launched("w4_pack");
}

extern "C" int evamx_w4_dequant(const evamx_w4_weight* w, float* out, evamx_stream_t stream)
{
    set_error("%s", "");
    if (!w4_weight_ok(w, "evamx_w4_dequant")) return EVAMX_EINVAL;
    if (!out) { set_error("evamx_w4_dequant: null pointer"); return EVAMX_EINVAL; }
    const size_t total = (size_t)w->count * w->n_out * w->n_in;
    w4_dequant_kernel<<<w4_grid(total), 256, 0, (hipStream_t)stream>>>(w4_mat(*w), W4_TILE_K / w->group, out, total);
    return launched("w4_dequant");
}
