// MXFP4 products (sm_100a): y[p, n] = sum_k q(x)[p, k] W[expert(p), n, k].
//
// A block forms 64 rows x 64 outputs from tiles of 32 columns (one scale a
// row), expanded to f32 in shared memory.
#include "iqk_host.cuh"
#include "iqk_mx.cuh"

namespace iqk {
namespace {

constexpr int kRows = 64, kOuts = 64;

struct ProductArgs {
    const uint8_t *codes, *scales;
    int64_t scale_stride, out_features, width;
    const uint8_t *xcodes, *xscales;
    int64_t pitch;
    int64_t pairs;
    const int32_t *hdr, *order;
    const int4 *tiles;
    void *y;
    int y_dtype;
};

__device__ __forceinline__ float scale_value(uint32_t byte) {
    if (byte == 255u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ float code_value(uint32_t code) {
    const float size = 0.5f * (float)((0xC8643210u >> (4 * (code & 7u))) & 15u);
    return (code & 8u) ? -size : size;
}

// Four values of a row's 32-column block into a column of the tile.
__device__ __forceinline__ void expand(const uint8_t *codes, const uint8_t *scales, int64_t width,
                                       int64_t stride, int64_t row, int k, int part,
                                       float (*tile)[kOuts + 1], int at, bool there) {
    const uint32_t w = there ? *reinterpret_cast<const uint32_t *>(codes + row * (width / 2) +
                                                                   k / 2 + part * 4)
                             : 0u;
    const float s = there ? scale_value(scales[row * stride + k / kMxBlock]) : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        tile[part * 8 + j][at] = there ? code_value((w >> (4 * j)) & 15u) * s : 0.f;
}

__device__ __forceinline__ void store(const ProductArgs &a, int64_t i, float v) {
    if (a.y_dtype == IQK_F32) static_cast<float *>(a.y)[i] = v;
    else if (a.y_dtype == IQK_F16) static_cast<__half *>(a.y)[i] = from_float<__half>(v);
    else static_cast<__nv_bfloat16 *>(a.y)[i] = from_float<__nv_bfloat16>(v);
}

__global__ void __launch_bounds__(256) mx_product_kernel(ProductArgs a) {
    __shared__ float xt[32][kRows + 1], wt[32][kOuts + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t nblocks = (a.out_features + kOuts - 1) / kOuts;
    const int64_t tiles = a.tiles ? a.hdr[1] : (a.pairs + kRows - 1) / kRows;
    if (a.tiles) {  // rows of pairs without an expert
        const int64_t tail = (a.pairs - a.hdr[2]) * a.out_features;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + tid; i < tail;
             i += (int64_t)gridDim.x * blockDim.x)
            store(a, a.order[a.hdr[2] + i / a.out_features] * a.out_features + i % a.out_features,
                  0.f);
    }
    for (int64_t item = blockIdx.x; item < tiles * nblocks; item += gridDim.x) {
        const int64_t t = item / nblocks, n0 = item % nblocks * kOuts;
        const int4 tile = a.tiles
            ? a.tiles[t]
            : make_int4(0, (int)(t * kRows), (int)min((int64_t)kRows, a.pairs - t * kRows), 0);
        float acc[4][4] = {};
        for (int k = 0; k < a.width; k += 32) {
            const int at = tid >> 2, part = tid & 3;
            expand(a.xcodes, a.xscales, a.width, a.pitch, (int64_t)tile.y + at, k, part, xt, at,
                   at < tile.z);
            expand(a.codes, a.scales, a.width, a.scale_stride,
                   (int64_t)tile.x * a.out_features + n0 + at, k, part, wt, at,
                   n0 + at < a.out_features);
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 32; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] += xt[kk][ty + 16 * i] * wt[kk][tx + 16 * j];
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty + 16 * i;
            if (r >= tile.z) continue;
            const int64_t pos = (int64_t)tile.y + r;
            const int64_t p = a.tiles ? a.order[pos] : pos;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + tx + 16 * j < a.out_features)
                    store(a, p * a.out_features + n0 + tx + 16 * j, acc[i][j]);
        }
    }
}

}  // namespace

MxLayout mx_layout(int64_t pairs, int64_t num_experts, int64_t width, int64_t out_features) {
    MxLayout L{};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += (bytes + 255) & ~size_t(255);
        return at;
    };
    L.cap = kRows;
    L.pitch = (width / kMxBlock + 15) / 16 * 16;
    L.max_tiles = (num_experts < pairs ? num_experts : pairs) + pairs / L.cap + 1;
    L.hdr = take(64);
    L.order = take(sizeof(int32_t) * (size_t)pairs);
    L.tiles = take(16 * (size_t)L.max_tiles);
    L.codes = take((size_t)pairs * (size_t)(width / 2));
    L.scales = take((size_t)pairs * (size_t)L.pitch);
    L.total = off;
    return L;
}

cudaError_t launch_mx_product(const MxProduct &p, cudaStream_t stream, int sms) {
    ProductArgs a{};
    a.codes = p.codes;
    a.scales = p.scales;
    a.scale_stride = p.scale_stride;
    a.out_features = p.out_features;
    a.width = p.width;
    a.xcodes = reinterpret_cast<const uint8_t *>(p.ws + p.L.codes);
    a.xscales = reinterpret_cast<const uint8_t *>(p.ws + p.L.scales);
    a.pitch = p.L.pitch;
    a.pairs = p.pairs;
    a.hdr = reinterpret_cast<const int32_t *>(p.ws + p.L.hdr);
    if (p.routed) {
        a.order = reinterpret_cast<const int32_t *>(p.ws + p.L.order);
        a.tiles = reinterpret_cast<const int4 *>(p.ws + p.L.tiles);
    }
    a.y = p.y;
    a.y_dtype = p.y_dtype;
    mx_product_kernel<<<(unsigned)(sms * 4), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace iqk
