// MXFP4 products (sm_100a, tcgen05 kind::mxf4 + TMEM):
//
//   y[p, n] = sum_b 2^(sx[p, b] + sw[n, b]) sum_{k in b} x[p, k] w[n, k]
//
// over blocks b of 32 columns, x and w E2M1 codes and sx, sw their block
// exponents, w the matrix of pair p's expert. The tensor core takes both
// operands as they lie in memory, codes and scales: nothing is expanded.
//
// The matrix is the MMA's M side (128 outputs) and the activations its N side
// (up to 128 rows), so a call with one token moves the matrix once and wastes
// only tensor-core columns that are idle anyway.
//
// Persistent, one CTA an SM, 12 warps:
//   warp 0      TMA producer: per unit of 512 columns the codes of 128 outputs
//               (two 128-byte-swizzle atoms) and of the tile's rows, and both
//               sides' scales (16 bytes a row)
//   warp 1      MMA issuer: eight K = 64 steps a unit
//   warp 2      tensor memory
//   warps 4-7   scale movers: the MMA reads scales from tensor memory, word
//               (row mod 32, row / 32) of each 128 columns, the same in all
//               four lane quarters; a row's 16 scale bytes are four such
//               words, so a mover lane reads 16 bytes a row group and stores
//               columns
//   warps 8-11  epilogue: tcgen05.ld, y stored (a warp's lanes are 32
//               consecutive outputs of one row)
// Accumulators and scale buffers are double-buffered.
//
// Work: item = (128 outputs, tile of rows). One matrix: rows innermost, so that
// it is read from memory once. Routed: outputs innermost, so that CTAs that run
// together read one matrix's rows next to each other (the other order strides
// by whole matrices and reads slower); an expert's next tile finds its matrix
// in L2. Full waves of items go to the CTAs in
// turn; what is left (under two waves) is cut into equal runs of units, and
// the parts of a shared item meet in f32 slots of the workspace: the last CTA
// to finish adds them in order, so results repeat bit for bit.
//
// Every wait is bounded (2 s): a wait that expires sets IQK_DEVERR_TIMEOUT and
// an abort flag that ends the others, copies in flight land, and tensor memory
// is freed before the CTA exits.
#include <cuda.h>

#include "iqk_host.cuh"
#include "iqk_mx.cuh"
#include "iqk_sync.cuh"

namespace iqk {
namespace {

using namespace dev;

constexpr int kThreads = 384;
constexpr int kProducer = 0, kIssuer = 1, kTmemWarp = 2, kMover0 = 4, kEpi0 = 8;
constexpr int kOuts = 128;              // outputs of an item (the MMA's M)
constexpr int kUnit = 512;              // columns of a pipeline stage
constexpr int kAtomA = kOuts * 128;     // one swizzle atom: 256 columns of 128 outputs
constexpr int kBoxes = 4;               // row boxes: 16, 32, 64, 128
constexpr int kMaxStages = 5;
constexpr int kSmemCap = 227 * 1024;
constexpr int kBarBytes = 256;
constexpr int kMaxCtas = 148;

// Shared memory of a stage: codes of the matrix, codes of the rows, scales.
__host__ __device__ constexpr int stage_bytes(int cap) {
    return 2 * kAtomA + 2 * cap * 128 + kOuts * 16 + cap * 16;
}
__host__ __device__ constexpr int stages_for(int cap) {
    const int n = (kSmemCap - 1024 - kBarBytes) / ((stage_bytes(cap) + 1023) & ~1023);
    return n < kMaxStages ? n : kMaxStages;
}

struct ProductArgs {
    int64_t out_features, width, pairs;
    int cap, stages;
    int32_t *hdr;
    const int32_t *order;  // null: one matrix, row p is pair p
    const int4 *tiles;
    int32_t *tickets;      // four per shared item, one for 32 outputs
    float *slots;          // [ctas, 2, cap, 128]
    void *y;
    int y_dtype;
};

struct Maps {
    CUtensorMap w, ws;                // matrix codes, scales
    CUtensorMap x[kBoxes], xs[kBoxes];  // rows' codes, scales; boxes of 16 << i rows
};

// The items of a call and how they are dealt to the CTAs.
struct Plan {
    uint32_t items, whole;   // whole: items dealt in full waves
    uint32_t tiles, nblocks, units;  // units of an item
    uint32_t all, runs;      // units of the shared items, CTAs that take a run of them
    uint32_t s0, s1;         // this CTA's run
    __device__ uint32_t start(uint32_t cta) const { return all * min(cta, runs) / runs; }
};

__device__ __forceinline__ Plan make_plan(const ProductArgs &a) {
    Plan p;
    const uint32_t ctas = gridDim.x;
    p.nblocks = (uint32_t)((a.out_features + kOuts - 1) / kOuts);
    p.tiles = a.tiles ? (uint32_t)a.hdr[1] : (uint32_t)((a.pairs + a.cap - 1) / a.cap);
    p.units = (uint32_t)((a.width + kUnit - 1) / kUnit);
    p.items = p.tiles * p.nblocks;
    const uint32_t waves = p.items / ctas;
    p.whole = p.items % ctas == 0 ? p.items : waves > 1 ? (waves - 1) * ctas : 0;
    // under two waves of items, at most 2^11 units each: 32 bits hold all * runs
    p.all = (p.items - p.whole) * p.units;
    p.runs = max(1u, min(ctas, p.all));
    p.s0 = p.start(blockIdx.x);
    p.s1 = p.start(blockIdx.x + 1);
    return p;
}

// One CTA's part of an item: units [u0, u1).
struct Part {
    uint32_t item;
    int u0, u1;
};

__device__ __forceinline__ bool part_of(const Plan &p, uint32_t i, Part &q) {
    const uint32_t mine = (p.whole + gridDim.x - 1 - blockIdx.x) / gridDim.x;
    if (i < mine) {
        q.item = blockIdx.x + i * gridDim.x;
        q.u0 = 0;
        q.u1 = (int)p.units;
        return true;
    }
    const uint32_t it = p.s0 / p.units + (i - mine), base = it * p.units;
    if (base >= p.s1 || p.s0 == p.s1) return false;
    q.item = p.whole + it;
    q.u0 = (int)(max(p.s0, base) - base);
    q.u1 = (int)(min(p.s1, base + p.units) - base);
    return true;
}

__device__ __forceinline__ int4 tile_of(const ProductArgs &a, const Plan &p, uint32_t item,
                                        int &out0) {
    if (a.tiles) {
        out0 = (int)(item % p.nblocks) * kOuts;
        return a.tiles[item / p.nblocks];
    }
    const uint32_t t = item % p.tiles;
    out0 = (int)(item / p.tiles) * kOuts;
    return make_int4(0, (int)(t * a.cap), (int)min((int64_t)a.cap, a.pairs - (int64_t)t * a.cap), 0);
}

// The smallest box that holds `rows`.
__device__ __forceinline__ int box_of(int rows) {
    return rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

__device__ __forceinline__ void store(const ProductArgs &a, int64_t i, float v) {
    if (a.y_dtype == IQK_F32) static_cast<float *>(a.y)[i] = v;
    else if (a.y_dtype == IQK_F16) static_cast<__half *>(a.y)[i] = from_float<__half>(v);
    else static_cast<__nv_bfloat16 *>(a.y)[i] = from_float<__nv_bfloat16>(v);
}

// Where the output row of the tile's row c + lane begins.
__device__ __forceinline__ int64_t row_base(const ProductArgs &a, const int4 &tile, int c,
                                            int lane) {
    if (c + lane >= tile.z) return 0;
    const int64_t pos = (int64_t)tile.y + c + lane;
    return (a.order ? a.order[pos] : pos) * a.out_features;
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int from) {
    return (int64_t)(((uint64_t)__shfl_sync(0xffffffffu, (uint32_t)((uint64_t)v >> 32), from) << 32) |
                     __shfl_sync(0xffffffffu, (uint32_t)(uint64_t)v, from));
}

// Columns [0, n) of v, each one row of y; lanes are 32 consecutive outputs from
// `out`. 16-bit outputs leave in pairs: lanes 2i and 2i + 1 swap halves, the
// even one stores both outputs of row j and the odd one of row j + 1 (4 bytes
// a lane; `pairs` says that rows of y begin on 4 bytes).
template <typename YT, int C>
__device__ __forceinline__ void store_columns(const ProductArgs &a, const float (&v)[C], int n,
                                              int64_t base, int lane, int out, bool pairs) {
    YT *y = static_cast<YT *>(a.y);
    const bool there = out < a.out_features;
    if (sizeof(YT) == 4 || !pairs) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int64_t at = shfl64(base, j);
            if (j < n && there) y[at + out] = from_float<YT>(v[j]);
        }
    } else {
        const int odd = lane & 1;
#pragma unroll
        for (int j = 0; j < C; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
            const int64_t at = shfl64(base, j + odd);
            struct __align__(4) Two { YT x, y; };
            const Two two{from_float<YT>(odd ? other : v[j]), from_float<YT>(odd ? v[j + 1] : other)};
            // out_features is even: an output and its neighbour exist together
            if (j + odd < n && there)
                *reinterpret_cast<Two *>(y + at + (out & ~1)) = two;
        }
    }
}

template <int C>
__device__ __forceinline__ void store_columns(const ProductArgs &a, const float (&v)[C], int n,
                                              int64_t base, int lane, int out, bool pairs) {
    if (a.y_dtype == IQK_F32) store_columns<float, C>(a, v, n, base, lane, out, pairs);
    else if (a.y_dtype == IQK_F16) store_columns<__half, C>(a, v, n, base, lane, out, pairs);
    else store_columns<__nv_bfloat16, C>(a, v, n, base, lane, out, pairs);
}

__global__ void __launch_bounds__(kThreads, 1)
mx_product_kernel(ProductArgs a, const __grid_constant__ Maps maps) {
    extern __shared__ char smem_raw[];
    // swizzle atoms repeat every 1024 bytes of shared memory
    const uint32_t raw = saddr(smem_raw);
    const uint32_t smem = (raw + 1023u) & ~1023u;
    const int S = a.stages, cap = a.cap;
    const uint32_t stage = (uint32_t)((stage_bytes(cap) + 1023) & ~1023);
    char *bars = smem_raw + (smem - raw) + S * stage;
    uint64_t *full = reinterpret_cast<uint64_t *>(bars);
    uint64_t *empty = full + kMaxStages;
    uint64_t *sready = empty + kMaxStages, *sfree = sready + 2;
    uint64_t *dfull = sfree + 2, *dempty = dfull + 2, *drain = dempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&sready[i], 4);
            bar_init(&sfree[i], 1);
            bar_init(&dfull[i], 1);
            bar_init(&dempty[i], 4);
        }
        bar_init(drain, 1);
        *abort_flag = 0;
        bar_fence_init();
    }
    if (warp == kTmemWarp) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
        tc_fence_before();
    }
    if (a.tiles) {  // rows of pairs without an expert
        const int64_t routed = a.hdr[2], tail = (a.pairs - routed) * a.out_features;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < tail;
             i += (int64_t)gridDim.x * blockDim.x)
            store(a, a.order[routed + i / a.out_features] * a.out_features + i % a.out_features,
                  0.f);
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: two accumulators of `cap`, then the scale buffers, 16 columns
    // a side and buffer (four words a row group, 128 rows)
    const uint32_t scale_col = tmem + 2 * cap;
    const Plan plan = make_plan(a);

    auto give_up = [&]() {
        if (!*abort_flag) {
            *abort_flag = 1;
            atomicOr(a.hdr, IQK_DEVERR_TIMEOUT);
        }
    };
    const uint32_t off_b = 2 * kAtomA, off_sa = off_b + 2 * cap * 128, off_sb = off_sa + kOuts * 16;

    if (warp == kProducer) {
        if (lane == 0) {
            int g = 0;
            bool ok = true;
            Part q;
            for (uint32_t i = 0; ok && !*abort_flag && part_of(plan, i, q); ++i) {
                int out0;
                const int4 tl = tile_of(a, plan, q.item, out0);
                const int box = box_of(tl.z), rows = 16 << box;
                const int row0 = (int)((int64_t)tl.x * a.out_features + out0);
                for (int u = q.u0; u < q.u1; ++u, ++g) {
                    const int s = g % S;
                    if (!bar_wait(&empty[s], ((uint32_t)(g / S) & 1u) ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    // the second half of the last unit may lie past the width
                    const int atoms = (int)min((int64_t)2, (a.width - (int64_t)u * kUnit + 255) / 256);
                    bar_expect_tx(&full[s], (uint32_t)(atoms * (kAtomA + rows * 128) +
                                                       (kOuts + rows) * 16));
                    const uint32_t st = smem + s * stage;
                    for (int t = 0; t < atoms; ++t) {
                        tma_2d(st + t * kAtomA, &maps.w, u * 256 + t * 128, row0, &full[s]);
                        tma_2d(st + off_b + t * rows * 128, &maps.x[box], u * 256 + t * 128, tl.y,
                               &full[s]);
                    }
                    tma_2d(st + off_sa, &maps.ws, u * 16, row0, &full[s]);
                    tma_2d(st + off_sb, &maps.xs[box], u * 16, tl.y, &full[s]);
                }
            }
            if (!ok) give_up();
            for (int d = 0; d < S && d < g; ++d) {  // every copy lands before the CTA exits
                const int gg = g - 1 - d;
                if (!bar_wait(&full[gg % S], (uint32_t)(gg / S) & 1u, nullptr)) give_up();
            }
        }
        __syncwarp();
    } else if (warp == kIssuer) {
        int g = 0, n = 0;
        bool ok = true;
        Part q;
        for (uint32_t i = 0; ok && part_of(plan, i, q); ++i, ++n) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int rows = 16 << box_of(tl.z);
            const int npad = (tl.z + 15) & ~15;
            const int acc = n & 1;
            ok = n < 2 || bar_wait_spin(&dempty[acc], ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            for (int u = q.u0; u < q.u1; ++u, ++g) {
                const int s = g % S, b = g & 1;
                ok = bar_wait_spin(&full[s], (uint32_t)(g / S) & 1u, abort_flag) &&
                     bar_wait_spin(&sready[b], (uint32_t)(g >> 1) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);  // elect.sync needs the warp converged
                if (!ok) break;
                tc_fence_after();
                const int steps = (int)min((int64_t)8, (a.width - (int64_t)u * kUnit + 63) / 64);
                if (elect_one()) {
                    const uint32_t st = smem + s * stage;
                    const uint32_t sa = scale_col + b * 32, sb = sa + 16;
                    for (int k = 0; k < steps; ++k) {
                        const uint32_t in = (uint32_t)(k & 3) * 32;
                        tc_mma_mxf4(tmem + acc * cap, sw128_desc(st + (k >> 2) * kAtomA + in),
                                    sw128_desc(st + off_b + (k >> 2) * rows * 128 + in),
                                    idesc_mxf4(kOuts, npad, (k & 1) * 2), sa + (k >> 1) * 4,
                                    sb + (k >> 1) * 4, (u > q.u0 || k > 0) ? 1u : 0u);
                    }
                    tc_commit(&empty[s]);
                    tc_commit(&sfree[b]);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (elect_one()) tc_commit(&dfull[acc]);
            __syncwarp();
        }
        if (!ok && lane == 0) give_up();
        __syncwarp();
        if (elect_one()) tc_commit(drain);  // every MMA ends before tensor memory is freed
        __syncwarp();
    } else if (warp >= kMover0 && warp < kMover0 + 4) {
        const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16;
        int g = 0;
        bool ok = true;
        Part q;
        for (uint32_t i = 0; ok && part_of(plan, i, q); ++i) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int rows = 16 << box_of(tl.z);
            for (int u = q.u0; u < q.u1; ++u, ++g) {
                const int s = g % S, b = g & 1;
                ok = bar_wait(&full[s], (uint32_t)(g / S) & 1u, abort_flag) &&
                     (g < 2 || bar_wait(&sfree[b], ((uint32_t)(g >> 1) & 1u) ^ 1u, abort_flag));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t st = smem + s * stage;
                const uint32_t dst = scale_col + quarter + b * 32;
                uint4 w[4], x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 32 * j + lane;
                    w[j] = lds128(st + off_sa + r * 16);
                    x[j] = r < rows ? lds128(st + off_sb + r * 16) : make_uint4(0u, 0u, 0u, 0u);
                }
                tmem_st4(dst + 0, w[0].x, w[1].x, w[2].x, w[3].x);
                tmem_st4(dst + 4, w[0].y, w[1].y, w[2].y, w[3].y);
                tmem_st4(dst + 8, w[0].z, w[1].z, w[2].z, w[3].z);
                tmem_st4(dst + 12, w[0].w, w[1].w, w[2].w, w[3].w);
                tmem_st4(dst + 16, x[0].x, x[1].x, x[2].x, x[3].x);
                tmem_st4(dst + 20, x[0].y, x[1].y, x[2].y, x[3].y);
                tmem_st4(dst + 24, x[0].z, x[1].z, x[2].z, x[3].z);
                tmem_st4(dst + 28, x[0].w, x[1].w, x[2].w, x[3].w);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&sready[b]);
            }
        }
        if (!ok) give_up();
    } else if (warp >= kEpi0) {
        const int quarter = warp & 3;
        const int r = 32 * quarter + lane;  // this thread's output of the item
        const bool pairs = a.out_features % 2 == 0 && reinterpret_cast<uintptr_t>(a.y) % 4 == 0;
        int n = 0;
        Part q;
        for (uint32_t i = 0; part_of(plan, i, q); ++i, ++n) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int acc = n & 1;
            const bool ok = bar_wait(&dfull[acc], (uint32_t)(n >> 1) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) {
                give_up();
                break;
            }
            tc_fence_after();
            const bool whole = (uint32_t)(q.u1 - q.u0) == plan.units;
            const uint32_t shared_item = q.item - plan.whole;
            // a run's first item has the run's first slot, its last the second
            const bool first = plan.s0 / plan.units == shared_item;
            float *slot = a.slots + ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * cap * kOuts;
            const uint32_t src = tmem + ((uint32_t)(32 * quarter) << 16) + acc * cap;
            for (int c = 0; c < tl.z; c += 16) {
                uint32_t d[2][8];
                const int here = min(16, tl.z - c);
                const int64_t base = whole ? row_base(a, tl, c, lane) : 0;
                tmem_ld8(src + c, d[0]);  // accumulators have a multiple of 16 columns
                tmem_ld8(src + c + 8, d[1]);
                tc_wait_ld();
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(d[j >> 3][j & 7]);
                if (whole) {
                    store_columns<16>(a, v, here, base, lane, out0 + r, pairs);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j < here) slot[(c + j) * kOuts + r] = v[j];
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&dempty[acc]);
            if (whole) continue;
            // A shared item: the CTA that finishes last adds every part, in order
            // (each warp for its 32 outputs: no warp waits for another).
            const uint32_t first_unit = shared_item * plan.units;
            auto owner = [&](uint32_t unit) {  // the CTA whose run holds the unit
                uint32_t o = unit * plan.runs / plan.all;
                while (plan.start(o + 1) <= unit) ++o;
                while (plan.start(o) > unit) --o;
                return o;
            };
            const uint32_t o0 = owner(first_unit), o1 = owner(first_unit + plan.units - 1);
            __threadfence();
            __syncwarp();
            uint32_t done = 0;
            if (lane == 0) done = (uint32_t)atomicAdd(&a.tickets[shared_item * 4 + quarter], 1);
            if (__shfl_sync(0xffffffffu, done, 0) != o1 - o0) continue;
            __threadfence();
            // the first owner's run may have begun in an earlier item
            const bool early = plan.start(o0) / plan.units != shared_item;
            for (int c = 0; c < tl.z; c += 8) {
                float v[8] = {};
                const int here = min(8, tl.z - c);
#pragma unroll 2
                for (uint32_t o = o0; o <= o1; ++o) {
                    const float *part = a.slots +
                        ((int64_t)o * 2 + (o == o0 && early ? 1 : 0)) * cap * kOuts + c * kOuts + r;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < here) v[j] += __ldcg(part + j * kOuts);
                }
                store_columns<8>(a, v, here, row_base(a, tl, c, lane), lane, out0 + r, pairs);
            }
        }
    }
    __syncthreads();
    if (warp == kTmemWarp) {
        if (lane == 0 && !bar_wait(drain, 0, nullptr)) give_up();
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

cudaError_t encode_rows(CUtensorMap *map, const void *base, uint64_t row_used, uint64_t rows,
                        uint64_t stride, uint32_t box_bytes, uint32_t box_rows, bool swizzle) {
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t err = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (err != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    const cuuint64_t dims[2] = {row_used, rows};
    const cuuint64_t strides[1] = {stride};
    const cuuint32_t box[2] = {box_bytes, box_rows};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult res = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base),
                                dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return res == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
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
    // Rows of a tile. Enough that an expert's rows mostly fit one tile, whose
    // matrix is then read once (an expert has `mean` rows or so), and fewer
    // while the call has less than an item for each SM: small tiles spread over
    // more SMs and have less to join.
    const int64_t nblocks = (out_features + kOuts - 1) / kOuts;
    const int64_t used = num_experts < pairs ? num_experts : pairs;
    const int64_t mean = pairs / num_experts;
    L.cap = num_experts == 1 || mean >= 24 ? 128 : mean >= 12 ? 64 : mean >= 4 ? 32 : 16;
    while (L.cap > 16 && (used + (pairs - used) / L.cap) * nblocks < kMaxCtas) L.cap /= 2;
    L.pitch = (width / kMxBlock + 15) / 16 * 16;
    L.max_tiles = (num_experts < pairs ? num_experts : pairs) + pairs / L.cap + 1;
    L.hdr = take(64);
    L.tickets = take(sizeof(int32_t) * 4 * 2 * kMaxCtas);
    L.order = take(sizeof(int32_t) * (size_t)pairs);
    L.place = take(sizeof(int32_t) * (size_t)((pairs + 3) / 4 * 4));
    L.tiles = take(16 * (size_t)L.max_tiles);
    L.codes = take((size_t)pairs * (size_t)(width / 2));
    L.scales = take((size_t)pairs * (size_t)L.pitch);
    L.slots = take(sizeof(float) * 2 * kMaxCtas * kOuts * (size_t)L.cap);
    L.total = off;
    return L;
}

cudaError_t launch_mx_product(const MxProduct &p, cudaStream_t stream, int sms) {
    ProductArgs a{};
    a.out_features = p.out_features;
    a.width = p.width;
    a.pairs = p.pairs;
    a.cap = p.L.cap;
    a.stages = stages_for(a.cap);
    a.hdr = reinterpret_cast<int32_t *>(p.ws + p.L.hdr);
    if (p.routed) {
        a.order = reinterpret_cast<const int32_t *>(p.ws + p.L.order);
        a.tiles = reinterpret_cast<const int4 *>(p.ws + p.L.tiles);
    }
    a.tickets = reinterpret_cast<int32_t *>(p.ws + p.L.tickets);
    a.slots = reinterpret_cast<float *>(p.ws + p.L.slots);
    a.y = p.y;
    a.y_dtype = p.y_dtype;
    Maps maps;
    const uint64_t rows = (uint64_t)(p.num_experts * p.out_features);
    const uint64_t code_row = (uint64_t)p.width / 2, scale_row = (uint64_t)p.width / kMxBlock;
    cudaError_t err = encode_rows(&maps.w, p.codes, code_row, rows, code_row, 128, kOuts, true);
    if (err == cudaSuccess)
        err = encode_rows(&maps.ws, p.scales, scale_row, rows, (uint64_t)p.scale_stride, 16, kOuts,
                          false);
    for (int i = 0; i < kBoxes && err == cudaSuccess; ++i) {
        err = encode_rows(&maps.x[i], p.ws + p.L.codes, code_row, (uint64_t)p.pairs, code_row, 128,
                          16u << i, true);
        if (err == cudaSuccess)
            err = encode_rows(&maps.xs[i], p.ws + p.L.scales, scale_row, (uint64_t)p.pairs,
                              (uint64_t)p.L.pitch, 16, 16u << i, false);
    }
    if (err != cudaSuccess) return err;
    const int smem = 1024 + a.stages * ((stage_bytes(a.cap) + 1023) & ~1023) + kBarBytes;
    static std::atomic<bool> attr_done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
    if (dev < 0 || !attr_done[dev].load()) {
        err = cudaFuncSetAttribute(mx_product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   kSmemCap);
        if (err != cudaSuccess) return err;
        if (dev >= 0) attr_done[dev].store(true);
    }
    const int grid = sms < kMaxCtas ? sms : kMaxCtas;
    mx_product_kernel<<<(unsigned)grid, kThreads, smem, stream>>>(a, maps);
    return cudaGetLastError();
}

}  // namespace iqk
