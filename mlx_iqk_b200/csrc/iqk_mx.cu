// MXFP4 quantisation and its inverse, and the entry points of the MXFP4
// products (sm_100a).
//
// A block is 32 consecutive values of a row. With m its largest magnitude,
//
//   scale = 2^max(floor(log2 m) - 2, -127),  code = round(v / scale) to E2M1
//
// so the largest value lands in [4, 8). Both steps are exact up to the one
// rounding: floor(log2 m) is m's exponent field, dividing by a power of two
// changes no digit, and cvt.rn.satfinite.e2m1x2 rounds to nearest even and
// holds what lies beyond 6 at 6. A NaN or an infinity has the largest exponent
// field, so the maximum of the magnitudes' bit patterns finds it, and the
// block's scale byte is 255 (NaN).
//
// Both kernels stream through memory. Quantisation gives a thread a whole block
// (half a block of f32): 64 bytes in four loads, one 16-byte store of codes and
// one scale. Four threads a block with a shuffled maximum took twice the
// instructions and wrote scales a quarter sector at a time (4096 x 4096 bf16:
// 14.3 us for 9.5 now, 4.4 TB/s).
#include <cooperative_groups.h>

#include <type_traits>

#include "iqk_host.cuh"
#include "iqk_mx.cuh"
#include "iqk_mx_block.cuh"

namespace iqk {
namespace {

// Row r of the output is row r of x; with `place`, row r of x goes to the rows
// place[r * copies ..] of its `copies` pairs (-1: none), so that a token's row
// is read and rounded once. That launch overlaps the sort that writes `place`:
// it waits for the sort after its first rows are read and rounded (`place` is
// volatile so that no load of it is moved above the wait). Block 0 clears the
// words that the product kernel counts in.
// I: an index type that holds rows * width / 16.
template <typename T, bool WIDE, typename I>
__global__ void __launch_bounds__(256)
mx_quantize_kernel(const T *__restrict__ x, I rows, I width, int64_t row_stride,
                   uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                   int64_t scale_stride, const volatile int32_t *place, int copies,
                   int32_t *__restrict__ zero, int zero_words) {
    grid_dep_launch();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < zero_words; i += blockDim.x) zero[i] = 0;
    constexpr int kShare = (int)sizeof(T) / 2;      // threads of a block
    constexpr int kValues = kMxBlock / kShare;      // values of a thread
    using Codes = typename std::conditional<kShare == 1, uint4, uint2>::type;
    const I per = width / kValues, all = rows * per, step = (I)gridDim.x * blockDim.x;
    I i = (I)blockIdx.x * blockDim.x + threadIdx.x;
    Walk<I> at(i, per, step);
    for (; i < all; i += step, at.next()) {
        const T *src = x + (int64_t)at.row * row_stride + (int64_t)at.col * kValues;
        Raw8<T> raw[kValues / 8];
#pragma unroll
        for (int j = 0; j < kValues / 8; ++j) load8<T, WIDE>(src + 8 * j, raw[j]);
        uint32_t amax = raw[0].peak();
#pragma unroll
        for (int j = 1; j < kValues / 8; ++j) amax = max(amax, raw[j].peak());
        // a block's two lanes stop together: `all` is even
        if (kShare == 2)
            amax = max(amax, __shfl_xor_sync(3u << (threadIdx.x & 30u), amax, 1));
        float inv;
        const uint32_t byte = scale_byte(amax, inv);
        Codes packed;
        uint32_t *word = reinterpret_cast<uint32_t *>(&packed);
#pragma unroll
        for (int j = 0; j < kValues / 8; ++j) {
            float v[8];
            raw[j].get(v);
            word[j] = codes8(v, inv);
        }
        if (place) grid_dep_wait();
        for (int j = 0; j < copies; ++j) {
            const int64_t to = place ? (int64_t)place[(int64_t)at.row * copies + j] : (int64_t)at.row;
            if (to < 0) continue;
            *reinterpret_cast<Codes *>(codes + to * (int64_t)(width / 2) +
                                       (int64_t)at.col * (kValues / 2)) = packed;
            if (at.col % kShare == 0)
                scales[to * scale_stride + (int64_t)(at.col / kShare)] = (uint8_t)byte;
        }
    }
    if (place) grid_dep_wait();  // a thread without items, too
}

// 2^(byte - 127); 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
    if (byte == 255u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Two codes of a byte to two values.
__device__ __forceinline__ float2 code_values(uint32_t byte) {
    uint32_t h;
    asm("{\n .reg .b8 b, z;\n mov.b32 {b, z, z, z}, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}\n"
        : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// A thread writes 16 bytes: four f32 or eight 16-bit values.
template <typename T, typename I>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                     int64_t scale_stride, I rows, I width, T *__restrict__ out) {
    constexpr int kN = 16 / (int)sizeof(T);
    const I per = width / kN, all = rows * per, step = (I)gridDim.x * blockDim.x;
    I i = (I)blockIdx.x * blockDim.x + threadIdx.x;
    Walk<I> at(i, per, step);
    for (; i < all; i += step, at.next()) {
        const uint32_t word = kN == 4 ? (uint32_t)reinterpret_cast<const uint16_t *>(codes)[i]
                                      : reinterpret_cast<const uint32_t *>(codes)[i];
        const float s = scale_value(
            scales[(int64_t)at.row * scale_stride + (int64_t)(at.col / (kMxBlock / kN))]);
        uint4 u;
        T *v = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
            const float2 f = code_values((word >> (8 * j)) & 0xffu);
            v[2 * j] = from_float<T>(f.x * s);
            v[2 * j + 1] = from_float<T>(f.y * s);
        }
        reinterpret_cast<uint4 *>(out)[i] = u;
    }
}

// Pairs by expert. A cluster of eight CTAs takes an eighth of the pairs each:
// it counts its pairs by expert (counting hands out the ranks, so that the
// second pass needs no atomics), reads the other CTAs' counts, and gives each
// of its pairs its place behind those of the CTAs before it. Pairs without an
// expert go to the tail of `order` and have place -1. CTA 0 cuts each expert's
// run into tiles of at most L.cap rows. Latency bounds it: one CTA took 14 us
// for 12288 pairs, most of it in shared-memory atomics.
//
// Each pair is a row of its own, so its tile changes no result as long as every
// item is summed whole; the atomics' order may then decide it. Where items can
// be shared (mx_may_join), tiles are cut at different columns and the row's f32
// sum depends on its tile: there ranks are handed out in the pairs' order
// (STABLE), so that a result repeats bit for bit; 12288 pairs take 4 us longer
// (of 167 us: 8192 columns, 2048 outputs, 64 experts).
constexpr int kSortCtas = 8;

template <bool STABLE>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(1024)
mx_sort_kernel(const int32_t *__restrict__ sel, int pairs, int num_experts, MxLayout L,
               char *ws) {
    grid_dep_launch();
    extern __shared__ int32_t cnt[];  // [num_experts + 1]: the last has no expert
    __shared__ int32_t warp_rows[32], warp_tiles[32], none_base;
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, wid = tid >> 5;
    const int rank = blockIdx.x;
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    int32_t *hdr = reinterpret_cast<int32_t *>(ws + L.hdr);
    int32_t *order = reinterpret_cast<int32_t *>(ws + L.order);
    int32_t *place = reinterpret_cast<int32_t *>(ws + L.place);
    int4 *tiles = reinterpret_cast<int4 *>(ws + L.tiles);
    for (int e = tid; e <= num_experts; e += nt) cnt[e] = 0;
    if (rank == 0)
        for (int i = tid; i < L.zeroed(); i += nt) hdr[i] = 0;
    const bool quads = (reinterpret_cast<uintptr_t>(sel) & 15) == 0;
    const int chunk = ((pairs + kSortCtas - 1) / kSortCtas + 3) / 4 * 4;
    const int p0 = rank * chunk, p1 = min(p0 + chunk, pairs);
    // the buckets of pairs p .. p + 3
    auto buckets = [&](int p, int (&e)[4]) {
        if (quads && p + 3 < p1) {
            const int4 v = *reinterpret_cast<const int4 *>(sel + p);
            e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = p + j < p1 ? sel[p + j] : -1;
        }
    };
    auto is_expert = [&](int e) { return e >= 0 && e < num_experts; };
    int stray = 0;
    __syncthreads();
    if constexpr (STABLE) {
        // A thread a pair: the warps find each pair's mates among their 32, and
        // warp 0 hands out the ranks, warp after warp.
        constexpr uint32_t kAll = 0xffffffffu;
        __shared__ int32_t bucket[1024];  // a pair's, then the rank of its first mate
        __shared__ uint32_t mates[1024];
        for (int p = p0; p < p1; p += 1024) {
            const int q = p + tid;
            const bool there = q < p1;
            const int v = there ? sel[q] : -1;
            const int b = is_expert(v) ? v : num_experts;
            stray |= b == num_experts && v != -1;
            const uint32_t same = __match_any_sync(kAll, b) & __ballot_sync(kAll, there);
            bucket[tid] = b;
            mates[tid] = there ? same : 0u;
            __syncthreads();
            for (int w = 0; wid == 0 && w < min(32, (p1 - p + 31) / 32); w += 8) {
                int e[8];
                uint32_t m[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    e[j] = bucket[32 * (w + j) + lane];
                    m[j] = mates[32 * (w + j) + lane];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int first = cnt[e[j]];
                    __syncwarp();
                    if (lane == __ffs(m[j]) - 1) cnt[e[j]] = first + __popc(m[j]);
                    bucket[32 * (w + j) + lane] = first;
                    __syncwarp();
                }
            }
            __syncthreads();
            if (there) place[q] = bucket[tid] + __popc(same & ((1u << lane) - 1u));
        }
    }
    for (int p = p0 + 4 * tid; !STABLE && p < p1; p += 4 * nt) {
        int e[4];
        buckets(p, e);
        int4 ranks = make_int4(0, 0, 0, 0);
        int *r = &ranks.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (p + j >= p1) continue;
            r[j] = atomicAdd(&cnt[is_expert(e[j]) ? e[j] : num_experts], 1);
            stray |= !is_expert(e[j]) && e[j] != -1;
        }
        *reinterpret_cast<int4 *>(place + p) = ranks;  // whole quads: see the layout
    }
    stray = __syncthreads_or(stray);
    cluster.sync();
    // exclusive sums of rows and tiles over the experts, `per` a thread
    const int per = (num_experts + nt - 1) / nt;
    const int e0 = min(tid * per, num_experts), e1 = min(e0 + per, num_experts);
    int rows = 0, made = 0, mine[4], total[4];  // per <= 4: at most 4096 experts
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        mine[k] = total[k] = 0;
        if (e0 + k >= e1) continue;
#pragma unroll
        for (int c = 0; c < kSortCtas; ++c) {
            const int n = cluster.map_shared_rank(cnt, c)[e0 + k];
            mine[k] += c < rank ? n : 0;
            total[k] += n;
        }
        rows += total[k];
        made += (total[k] + L.cap - 1) / L.cap;
    }
    if (tid == 0) {
        int n = 0;
        for (int c = 0; c < rank; ++c) n += cluster.map_shared_rank(cnt, c)[num_experts];
        none_base = n;
    }
    int at = rows, tile = made;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, at, o), b = __shfl_up_sync(0xffffffffu, tile, o);
        if (lane >= o) at += a, tile += b;
    }
    if (lane == 31) warp_rows[wid] = at, warp_tiles[wid] = tile;
    cluster.sync();  // every CTA has read the counts: they become cursors
    at -= rows, tile -= made;
    int all_rows = 0, all_tiles = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
        if (w == wid) at += all_rows, tile += all_tiles;
        all_rows += warp_rows[w], all_tiles += warp_tiles[w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (e0 + k >= e1) continue;
        if (rank == 0)
            for (int i = 0; i < total[k]; i += L.cap)
                tiles[tile++] = make_int4(e0 + k, at + i, min(L.cap, total[k] - i), 0);
        cnt[e0 + k] = at + mine[k];
        at += total[k];
    }
    if (tid == 0) {
        cnt[num_experts] = all_rows + none_base;
        if (rank == 0) {
            hdr[1] = all_tiles;
            hdr[2] = all_rows;
        }
    }
    __syncthreads();
    // after the clearing of hdr: the cluster has synchronised twice since
    if (tid == 0 && stray) atomicOr(hdr, IQK_DEVERR_EXPERT);
    for (int p = p0 + 4 * tid; p < p1; p += 4 * nt) {
        int e[4];
        buckets(p, e);
        int4 to = *reinterpret_cast<const int4 *>(place + p);
        int *r = &to.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (p + j >= p1) continue;
            r[j] += cnt[is_expert(e[j]) ? e[j] : num_experts];
            order[r[j]] = p + j;
            if (!is_expert(e[j])) r[j] = -1;
        }
        *reinterpret_cast<int4 *>(place + p) = to;
    }
}

// Blocks of a streaming kernel: eight an SM, fewer for fewer items.
unsigned stream_blocks(int64_t items, int sms) {
    const int64_t want = (items + 255) / 256, most = (int64_t)sms * 8;
    return (unsigned)(want < most ? want : most);
}

size_t element(int dtype) { return dtype == IQK_F32 ? 4 : 2; }

int check_matrix(const uint8_t *codes, const uint8_t *scales, int64_t scale_stride, int64_t rows,
                 int64_t width) {
    if (width <= 0 || width % kMxBlock || width > (1 << 20)) return IQK_ERR_GEOMETRY;
    if (rows < 0 || rows > ((int64_t)1 << 31) - 1) return IQK_ERR_GEOMETRY;
    if (scale_stride < width / kMxBlock || scale_stride % 16) return IQK_ERR_ALIGNMENT;
    if (rows == 0) return IQK_OK;
    if (!codes || !scales) return IQK_ERR_ARGUMENT;
    if (!aligned(codes, 16) || !aligned(scales, 16)) return IQK_ERR_ALIGNMENT;
    return IQK_OK;
}

int check_rows(const void *x, int dtype, int64_t rows, int64_t width, int64_t row_stride) {
    if (!dtype_ok(dtype)) return IQK_ERR_ARGUMENT;
    if (rows < 0 || rows > ((int64_t)1 << 31) - 1) return IQK_ERR_GEOMETRY;
    if (rows > 1 && row_stride < width && row_stride != 0) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    if (!x) return IQK_ERR_ARGUMENT;
    if (!aligned(x, element(dtype))) return IQK_ERR_ALIGNMENT;
    return IQK_OK;
}

// The product kernel counts its items in 32 bits.
bool mx_items_ok(const MxProduct &p) {
    return p.L.max_tiles * ((p.out_features + p.L.outs - 1) / p.L.outs) < (int64_t)1 << 31;
}

}  // namespace

cudaError_t launch_mx_quantize(const void *x, int dtype, int64_t rows, int64_t width,
                               int64_t row_stride, uint8_t *codes, uint8_t *scales,
                               int64_t scale_stride, const int32_t *place, int copies,
                               int32_t *zero, int zero_words,
                               cudaStream_t stream, int sms) {
    const unsigned blocks = stream_blocks(rows * width * (int64_t)element(dtype) / 64, sms);
    const bool wide = aligned(x, 16) && row_stride * (int64_t)element(dtype) % 16 == 0;
    const bool small = rows * (width / 16) < (int64_t)1 << 31;
    PdlLaunch pl(blocks, 256, 0, stream);
    if (!place) pl.cfg.numAttrs = 0;  // what precedes it may have written x
    cudaError_t err;
#define IQK_QI(T, W, I)                                                                         \
    err = cudaLaunchKernelEx(&pl.cfg, mx_quantize_kernel<T, W, I>, static_cast<const T *>(x),   \
                             (I)rows, (I)width, row_stride, codes, scales, scale_stride, place, \
                             copies, zero, zero_words)
#define IQK_Q(T)                                        \
    do {                                                \
        if (wide && small) IQK_QI(T, true, uint32_t);   \
        else if (small) IQK_QI(T, false, uint32_t);     \
        else if (wide) IQK_QI(T, true, uint64_t);       \
        else IQK_QI(T, false, uint64_t);                \
    } while (0)
    if (dtype == IQK_F32) IQK_Q(float);
    else if (dtype == IQK_F16) IQK_Q(__half);
    else IQK_Q(__nv_bfloat16);
#undef IQK_QI
#undef IQK_Q
    return err;
}

}  // namespace iqk

using namespace iqk;

extern "C" {

int iqk_mx_quantize(const void *x, int dtype, int64_t rows, int64_t width, int64_t row_stride,
                    uint8_t *codes, uint8_t *scales, int64_t scale_stride, iqk_stream_t stream) {
    int st = check_matrix(codes, scales, scale_stride, rows, width);
    if (st == IQK_OK) st = check_rows(x, dtype, rows, width, row_stride);
    if (st != IQK_OK || rows == 0) return st;
    return cuda_status(launch_mx_quantize(x, dtype, rows, width, row_stride, codes, scales,
                                          scale_stride, nullptr, 1, nullptr, 0,
                                          reinterpret_cast<cudaStream_t>(stream),
                                          num_sms_current()));
}

int iqk_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t scale_stride,
                      int64_t rows, int64_t width, void *out, int out_dtype,
                      iqk_stream_t stream) {
    const int st = check_matrix(codes, scales, scale_stride, rows, width);
    if (st != IQK_OK) return st;
    if (!dtype_ok(out_dtype)) return IQK_ERR_ARGUMENT;
    if (rows == 0) return IQK_OK;
    if (!out) return IQK_ERR_ARGUMENT;
    if (!aligned(out, 16)) return IQK_ERR_ALIGNMENT;
    const int64_t items = rows * width * (int64_t)element(out_dtype) / 16;
    const unsigned blocks = stream_blocks(items, num_sms_current());
    const bool small = items < (int64_t)1 << 31;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define IQK_DI(T, I)                                                                   \
    mx_dequantize_kernel<T, I><<<blocks, 256, 0, s>>>(codes, scales, scale_stride, (I)rows, \
                                                      (I)width, static_cast<T *>(out))
#define IQK_D(T)                      \
    do {                              \
        if (small) IQK_DI(T, uint32_t); \
        else IQK_DI(T, uint64_t);     \
    } while (0)
    if (out_dtype == IQK_F32) IQK_D(float);
    else if (out_dtype == IQK_F16) IQK_D(__half);
    else IQK_D(__nv_bfloat16);
#undef IQK_DI
#undef IQK_D
    return cuda_status(cudaGetLastError());
}

size_t iqk_mx_workspace_bytes(int64_t pairs, int64_t num_experts, int64_t width,
                              int64_t out_features) {
    if (pairs < 0 || pairs > (1 << 24) || num_experts <= 0 || num_experts > 4096 || width <= 0 ||
        width % kMxBlock || width > (1 << 20) || out_features <= 0)
        return 0;
    return mx_layout(pairs, num_experts, width, out_features).total;
}

int iqk_mx_linear(const void *x, int x_dtype, int64_t rows, int64_t row_stride,
                  const uint8_t *codes, const uint8_t *scales, int64_t scale_stride,
                  int64_t out_features, int64_t width, void *y, int y_dtype, void *workspace,
                  size_t workspace_bytes, iqk_stream_t stream) {
    if (out_features <= 0) return IQK_ERR_GEOMETRY;
    int st = check_matrix(codes, scales, scale_stride, out_features, width);
    if (st == IQK_OK) st = check_rows(x, x_dtype, rows, width, row_stride);
    if (st != IQK_OK) return st;
    if (!dtype_ok(y_dtype)) return IQK_ERR_ARGUMENT;
    if (rows > (1 << 24)) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    if (!y || !workspace) return IQK_ERR_ARGUMENT;
    if (!aligned(y, element(y_dtype)) || !aligned(workspace, 256)) return IQK_ERR_ALIGNMENT;
    MxProduct p{codes, scales, scale_stride, out_features, width, rows, 1,
                static_cast<char *>(workspace), mx_layout(rows, 1, width, out_features), false,
                y, y_dtype};
    if (workspace_bytes < p.L.total) return IQK_ERR_WORKSPACE;
    if (!mx_items_ok(p)) return IQK_ERR_GEOMETRY;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int sms = num_sms_current();
    cudaError_t err = launch_mx_quantize(x, x_dtype, rows, width, row_stride,
                             reinterpret_cast<uint8_t *>(p.ws + p.L.codes),
                             reinterpret_cast<uint8_t *>(p.ws + p.L.scales), p.L.pitch, nullptr, 1,
                             reinterpret_cast<int32_t *>(p.ws + p.L.hdr), p.L.zeroed(), s, sms);
    if (err != cudaSuccess) return cuda_status(err);
    return cuda_status(launch_mx_product(p, s, sms));
}

int iqk_mx_routed(const void *x, int x_dtype, int64_t x_rows, int64_t row_stride,
                  const int32_t *sel, int64_t pairs, const uint8_t *codes,
                  const uint8_t *scales, int64_t scale_stride, int64_t num_experts,
                  int64_t out_features, int64_t width, void *y, int y_dtype, void *workspace,
                  size_t workspace_bytes, iqk_stream_t stream) {
    if (out_features <= 0 || num_experts <= 0 || num_experts > 4096) return IQK_ERR_GEOMETRY;
    if (out_features > ((int64_t)1 << 31) / num_experts) return IQK_ERR_GEOMETRY;
    int st = check_matrix(codes, scales, scale_stride, num_experts * out_features, width);
    if (st == IQK_OK) st = check_rows(x, x_dtype, x_rows, width, row_stride);
    if (st != IQK_OK) return st;
    if (!dtype_ok(y_dtype)) return IQK_ERR_ARGUMENT;
    if (pairs < 0 || pairs > (1 << 24)) return IQK_ERR_GEOMETRY;
    if (pairs == 0) return IQK_OK;
    if (x_rows <= 0 || pairs % x_rows) return IQK_ERR_GEOMETRY;
    if (!y || !workspace || !sel) return IQK_ERR_ARGUMENT;
    if (!aligned(y, element(y_dtype)) || !aligned(workspace, 256) || !aligned(sel, 4))
        return IQK_ERR_ALIGNMENT;
    MxProduct p{codes, scales, scale_stride, out_features, width, pairs, num_experts,
                static_cast<char *>(workspace),
                mx_layout(pairs, num_experts, width, out_features), true, y, y_dtype};
    if (workspace_bytes < p.L.total) return IQK_ERR_WORKSPACE;
    if (!mx_items_ok(p)) return IQK_ERR_GEOMETRY;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int sms = num_sms_current();
    const size_t counts = sizeof(int32_t) * (size_t)(num_experts + 1);
    if (mx_may_join(width))
        mx_sort_kernel<true><<<kSortCtas, 1024, counts, s>>>(sel, (int)pairs, (int)num_experts,
                                                             p.L, p.ws);
    else
        mx_sort_kernel<false><<<kSortCtas, 1024, counts, s>>>(sel, (int)pairs, (int)num_experts,
                                                              p.L, p.ws);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return cuda_status(err);
    err = launch_mx_quantize(x, x_dtype, x_rows, width, row_stride,
                             reinterpret_cast<uint8_t *>(p.ws + p.L.codes),
                             reinterpret_cast<uint8_t *>(p.ws + p.L.scales), p.L.pitch,
                             reinterpret_cast<const int32_t *>(p.ws + p.L.place),
                             (int)(pairs / x_rows), nullptr, 0, s, sms);
    if (err != cudaSuccess) return cuda_status(err);
    return cuda_status(launch_mx_product(p, s, sms));
}

int iqk_mx_read_error(const void *workspace, int32_t *flags, iqk_stream_t stream) {
    if (!workspace || !flags) return IQK_ERR_ARGUMENT;
    *flags = 0;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int32_t word[4] = {};
    cudaError_t err = cudaMemcpyAsync(word, workspace, sizeof(word), cudaMemcpyDeviceToHost, s);
    if (err == cudaSuccess) err = cudaStreamSynchronize(s);
    if (err == cudaSuccess) *flags = word[0] | word[3];
    return cuda_status(err);
}

int iqk_mx_error_word(int32_t **word) {
    if (!word) return IQK_ERR_ARGUMENT;
    return cuda_status(mx_error_word(word));
}

int iqk_mx_take_errors(int32_t *flags, iqk_stream_t stream) {
    if (!flags) return IQK_ERR_ARGUMENT;
    *flags = 0;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int32_t *word = nullptr, value = 0;
    cudaError_t err = mx_error_word(&word);
    if (err == cudaSuccess)
        err = cudaMemcpyAsync(&value, word, sizeof(value), cudaMemcpyDeviceToHost, s);
    if (err == cudaSuccess) err = cudaStreamSynchronize(s);
    if (err == cudaSuccess && value) err = cudaMemsetAsync(word, 0, sizeof(value), s);
    if (err == cudaSuccess) *flags = value;
    return cuda_status(err);
}

size_t iqk_mx_few_state_bytes(void) { return mx_few_state_bytes(1 << 20); }

size_t iqk_mx_few_state_bytes_for(int64_t width) { return mx_few_state_bytes(width); }

int iqk_mx_few_fits(int64_t pairs, int64_t num_experts, int64_t out_features, int64_t width,
                    int routed) {
    return pairs > 0 && num_experts > 0 && out_features > 0 && width > 0 &&
           mx_few_fits(pairs, num_experts, out_features, width, routed != 0);
}

int iqk_mx_few(const void *x, int x_dtype, int64_t x_rows, int64_t row_stride, const int32_t *sel,
               int64_t pairs, const uint8_t *codes, const uint8_t *scales, int64_t scale_stride,
               int64_t num_experts, int64_t out_features, int64_t width, void *y, int y_dtype,
               void *state, size_t state_bytes, iqk_stream_t stream) {
    if (out_features <= 0 || num_experts <= 0 || num_experts > 4096) return IQK_ERR_GEOMETRY;
    if (!sel && num_experts != 1) return IQK_ERR_GEOMETRY;
    if (out_features > ((int64_t)1 << 31) / num_experts) return IQK_ERR_GEOMETRY;
    int st = check_matrix(codes, scales, scale_stride, num_experts * out_features, width);
    if (st == IQK_OK) st = check_rows(x, x_dtype, x_rows, width, row_stride);
    if (st != IQK_OK) return st;
    if (!dtype_ok(y_dtype)) return IQK_ERR_ARGUMENT;
    if (pairs < 0 || !mx_few_fits(pairs, num_experts, out_features, width, sel != nullptr))
        return IQK_ERR_GEOMETRY;
    if (pairs == 0) return IQK_OK;
    if (x_rows <= 0 || pairs % x_rows || (!sel && pairs != x_rows)) return IQK_ERR_GEOMETRY;
    if (!y || !state) return IQK_ERR_ARGUMENT;
    if (!aligned(y, element(y_dtype)) || !aligned(state, 256) || !aligned(sel, 4))
        return IQK_ERR_ALIGNMENT;
    if (state_bytes < mx_few_state_bytes(width)) return IQK_ERR_WORKSPACE;
    const MxFew p{x, x_dtype, x_rows, row_stride, sel, pairs, codes, scales, scale_stride,
                  num_experts, out_features, width, y, y_dtype, static_cast<char *>(state)};
    return cuda_status(launch_mx_few(p, reinterpret_cast<cudaStream_t>(stream),
                                     num_sms_current()));
}

}  // extern "C"
