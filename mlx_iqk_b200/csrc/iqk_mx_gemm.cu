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
// Persistent, one CTA an SM, 16 warps; a unit is 512 columns, a stage half of it:
//   warp 0      TMA producer: per stage the codes of 128 outputs and of the
//               tile's rows, a 128-byte-swizzle atom each
//   warp 1      MMA issuer: four K = 64 steps a stage
//   warp 2      tensor memory; zeros to rows of pairs without an expert
//   warp 3      TMA of both sides' scales, 16 bytes a row and unit, on a ring of
//               their own: they run ahead of the codes, so that a unit's scales
//               are in tensor memory before its codes have come
//   warps 4-7   scale movers: the MMA reads scales from tensor memory, word
//               (row mod 32, row / 32) of each 128 columns, the same in all
//               four lane quarters; a row's 16 scale bytes are four such
//               words, so a mover lane reads 16 bytes a row group and stores
//               columns
//   warps 8-11  epilogue: tcgen05.ld, y stored (a warp's lanes are 32
//               consecutive outputs of one row)
//   warps 12-15 the second half of the tile's rows in the epilogue. Few rows:
//               activations instead: the rows' 512 columns read from x,
//               rounded and written where TMA would have put them, so that
//               such a call is one launch; each CTA also sorts its (at most
//               64) pairs by itself. With up to 4 rows a tile each warp takes
//               every fourth unit, so that four units' loads are under way (a
//               quarter off 8 tokens' down projection); with more, the warps
//               share each unit (a sixth off a call of 37 rows)
// Accumulators are double-buffered, scale buffers up to four deep.
//
// What bounds it. A call whose matrix comes from HBM runs at the copy rate: the
// head product, 129280 x 4096 for one token, takes 49 us (281.6 MB, 43 at the
// copy rate, after 4.5 us of start), a routed prefill 192 us (1.21 GB). One
// whose matrix stays in L2 is bound by what an SM can load, 64 bytes a clock:
// 4096 x 4096 x 8192 takes 74 us (3.7 PFLOP/s), its copies alone 59. One warp's
// chain of dependent instructions issues every product, so what it waits for
// paces the kernel: with whole units as stages, of which three fit, and three
// barriers a unit that case took 95 us.
//
// Work: item = (128 outputs, tile of rows); a call of few items takes 64 or 32
// outputs to an item and leaves the MMA's other rows unused, which spreads the
// matrix over more SMs. One matrix: rows innermost, so that it is read from
// memory once. Routed: outputs innermost, so that CTAs that run together read
// one matrix's rows next to each other (the other order strides by whole
// matrices: a tenth slower in a prefill); an expert's next tile finds its
// matrix in L2. The CTAs take items in turn. Where the last round would leave many of
// them idle over a wide matrix, its items are cut into equal runs of units, and
// the parts of an item meet in f32 slots of the workspace: the last CTA to
// finish adds them in order. Routed pairs of such widths are sorted in their own
// order, so that a pair is in the same tile each time: results repeat bit for bit.
//
// The kernel is a programmatic dependent launch: barriers and tensor memory are
// set up while the kernel before it drains (1.5 us off each call in a row).
//
// Every wait is bounded (2 s): a wait that expires sets IQK_DEVERR_TIMEOUT and
// an abort flag that ends the others, copies in flight land, and tensor memory
// is freed before the CTA exits.
#include <cuda.h>

#include <type_traits>

#include "iqk_host.cuh"
#include "iqk_mx.cuh"
#include "iqk_mx_block.cuh"
#include "iqk_sync.cuh"

namespace iqk {
namespace {

using namespace dev;

constexpr int kThreads = 512;
constexpr int kProducer = 0, kIssuer = 1, kTmemWarp = 2, kScaleWarp = 3, kMover0 = 4, kEpi0 = 8,
              kRound0 = 12;
constexpr int kOuts = 128;              // outputs of an item at most (the MMA's M)
constexpr int kUnit = 512;              // columns of a 16-byte row of scales
constexpr int kStageK = 256;            // columns of a stage: one swizzle atom a side
constexpr int kScales = 4;              // scale slots, in shared and in tensor memory
constexpr int kBoxes = 4;               // row boxes: 16, 32, 64, 128
constexpr int kMaxUnits = 12;           // units in flight: two stages each
constexpr int kSmemCap = 227 * 1024;
constexpr int kBarBytes = 640;
constexpr int kFewCap = 16, kFewPairs = 64;          // one launch: rows of a tile, routed pairs
constexpr int kFewTable = kFewPairs * (16 + 2 * 4 * kFewCap);  // tiles; pairs, rows of x
constexpr int kMaxCtas = 148;
constexpr uint32_t kSaved = 14;

// Shared memory: stages (codes of the outputs and of the rows), scale slots.
__host__ __device__ constexpr int stage_bytes(int cap, int outs) { return (outs + cap) * 128; }
__host__ __device__ constexpr int slot_bytes(int cap, int outs) { return (outs + cap) * 16; }
// The MMA reads 128 outputs of a stage whatever an item has: what follows the
// last stage must be shared memory too.
__host__ __device__ constexpr int spare_bytes(int cap, int outs) {
    return kOuts * 128 > stage_bytes(cap, outs) ? kOuts * 128 - stage_bytes(cap, outs) : 0;
}
__host__ __device__ constexpr int smem_fixed(int cap, int outs) {
    return 1024 + kBarBytes + kFewTable + spare_bytes(cap, outs) + kScales * slot_bytes(cap, outs);
}
__host__ __device__ constexpr int units_for(int cap, int outs) {
    const int n = (kSmemCap - smem_fixed(cap, outs)) / (2 * stage_bytes(cap, outs));
    return n < kMaxUnits ? n : kMaxUnits;
}

struct ProductArgs {
    int64_t out_features, width, pairs;
    int cap, outs, units;  // units: in flight
    int32_t *hdr;
    const int32_t *order;  // null: one matrix, row p is pair p
    const int4 *tiles;
    int32_t *tickets;      // per shared item: 32 outputs x half of the rows
    float *slots;          // [ctas, 2, cap, 128]
    void *y;
    int y_dtype;
    // few rows: the activations themselves, row p / per_row for pair p
    const void *x;
    int64_t x_stride;
    const int32_t *sel;    // null: one matrix
    int per_row, experts, wide;
    int spread;            // the four rounding warps share each unit, else take turns
};

struct MatrixMaps {
    CUtensorMap w, ws;  // matrix codes, scales
};
struct Maps : MatrixMaps {
    CUtensorMap x[kBoxes], xs[kBoxes];  // rows' codes, scales; boxes of 16 << i rows
};
template <bool FEW> using MapsOf = typename std::conditional<FEW, MatrixMaps, Maps>::type;

// The items of a call and how they are dealt to the CTAs.
struct Plan {
    uint32_t items, whole;   // whole: items dealt in full waves
    uint32_t tiles, nblocks, units;  // units of an item
    uint32_t all, runs;      // units of the shared items, CTAs that take a run of them
    uint32_t s0, s1;         // this CTA's run
    __device__ uint32_t start(uint32_t cta) const { return all * min(cta, runs) / runs; }
};

// join: items may be shared.
__device__ __forceinline__ Plan make_plan(const ProductArgs &a, int routed_tiles, bool join) {
    Plan p;
    const uint32_t ctas = gridDim.x;
    p.nblocks = (uint32_t)((a.out_features + a.outs - 1) / a.outs);
    p.tiles = a.tiles ? (uint32_t)routed_tiles : (uint32_t)((a.pairs + a.cap - 1) / a.cap);
    p.units = (uint32_t)((a.width + kUnit - 1) / kUnit);
    p.items = p.tiles * p.nblocks;
    // The last round's items are shared when that saves kSaved units or more:
    // joining parts costs 4 to 8 us (a fence, a counter and the sums), a unit
    // 0.4 us for a CTA that has the memory to itself. A decode step's 96 items
    // of 8 units were done after 13 us when cut to fill all SMs, after 10 whole.
    const uint32_t rest = p.items % ctas, run = (rest * p.units + ctas - 1) / ctas;
    p.whole = !join || p.units - run < kSaved ? p.items : p.items - rest;
    // fewer items than CTAs, at most 2^11 units each: 32 bits hold all * runs
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
        out0 = (int)(item % p.nblocks) * a.outs;
        return a.tiles[item / p.nblocks];
    }
    const uint32_t t = item % p.tiles;
    out0 = (int)(item / p.tiles) * a.outs;
    return make_int4(0, (int)(t * a.cap), (int)min((int64_t)a.cap, a.pairs - (int64_t)t * a.cap), 0);
}

// The smallest box that holds the tile's rows; one matrix: the box of a full
// tile, which the last one's rows beyond the activations read as zeros.
__device__ __forceinline__ int box_of(const ProductArgs &a, const int4 &tile) {
    const int rows = a.tiles ? tile.z : a.cap;
    return rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
}

// A place in a ring of units or scale slots.
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int size) {
        if (++s == size) {
            s = 0;
            phase ^= 1u;
        }
    }
};

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

// Zeros to row p of y, by one warp, 16 bytes a lane where they are aligned.
__device__ __forceinline__ void zero_row(const ProductArgs &a, int64_t p, int lane) {
    const int64_t item = a.y_dtype == IQK_F32 ? 4 : 2;
    char *row = static_cast<char *>(a.y) + p * a.out_features * item;
    const int64_t bytes = a.out_features * item;
    const int64_t head = min(bytes, (int64_t)(-reinterpret_cast<intptr_t>(row) & 15));
    const int64_t body = (bytes - head) / 16;
    for (int64_t i = 2 * lane; i < head; i += 64) *reinterpret_cast<uint16_t *>(row + i) = 0;
    for (int64_t i = lane; i < body; i += 32)
        reinterpret_cast<uint4 *>(row + head)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int64_t i = head + 16 * body + 2 * lane; i < bytes; i += 64)
        *reinterpret_cast<uint16_t *>(row + i) = 0;
}

// Few pairs, sorted by one warp (lane l: pairs l and l + 32): a pair's rank is
// the number of earlier pairs of its expert, every 16th rank opens a tile, and
// the pair's row is its rank in the tile. Returns the tiles; `bad` says that an
// index is neither an expert nor -1.
__device__ __forceinline__ int sort_few(const ProductArgs &a, int lane, int4 *tiles,
                                        int32_t *pairs, int32_t *rows, bool &bad) {
    constexpr uint32_t kAll = 0xffffffffu;
    int e[2], rank[2], count[2], lead[2] = {0, 0};
    bool stray = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int p = lane + 32 * h;
        e[h] = p < a.pairs ? a.sel[p] : -1;
        if (e[h] < 0 || e[h] >= a.experts) {
            stray |= e[h] != -1;
            e[h] = -1;
        }
    }
    bad = __any_sync(kAll, stray);
    const bool two = a.pairs > 32;
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t same = __match_any_sync(kAll, e[h]);
        rank[h] = __popc(same & below);
        count[h] = __popc(same);
    }
    if (two) {
#pragma unroll 8
        for (int q = 0; q < 32; ++q) {
            const int other0 = __shfl_sync(kAll, e[0], q), other1 = __shfl_sync(kAll, e[1], q);
            const int in0 = other0 == e[1], in1 = other1 == e[0];
            rank[1] += in0;
            count[1] += in0;
            count[0] += in1;
        }
    }
    const uint32_t m0 = __ballot_sync(kAll, e[0] >= 0 && rank[0] % kFewCap == 0);
    const uint32_t m1 = __ballot_sync(kAll, e[1] >= 0 && rank[1] % kFewCap == 0);
    // the pair that opened this one's tile
    const int from[2] = {rank[0] & -kFewCap, rank[1] & -kFewCap};
#pragma unroll 8
    for (int q = 0; q < 32; ++q) {
        const int oe = __shfl_sync(kAll, e[0], q), orank = __shfl_sync(kAll, rank[0], q);
        if (oe == e[0] && orank == from[0]) lead[0] = q;
        if (oe == e[1] && orank == from[1]) lead[1] = q;
    }
    if (two) {
#pragma unroll 8
        for (int q = 0; q < 32; ++q) {
            const int oe = __shfl_sync(kAll, e[1], q), orank = __shfl_sync(kAll, rank[1], q);
            if (oe == e[1] && orank == from[1]) lead[1] = q + 32;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (e[h] < 0) continue;
        const int p = lane + 32 * h;
        const uint32_t under = (1u << (lead[h] & 31)) - 1u;
        const int tile = lead[h] < 32 ? __popc(m0 & under) : __popc(m0) + __popc(m1 & under);
        const int at = tile * kFewCap + rank[h] % kFewCap;
        if (lead[h] == p)
            tiles[tile] = make_int4(e[h], tile * kFewCap, min(kFewCap, count[h] - rank[h]), 0);
        pairs[at] = p;
        rows[at] = p / a.per_row;
    }
    return __popc(m0) + __popc(m1);
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

// Error bits of every product on this device, beside those of a call's own
// workspace or state, which may be gone before anyone reads them.
__device__ int32_t device_errors;

// FEW: activations of type XT, rounded in the kernel; else from the workspace.
template <bool FEW, typename XT>
__global__ void __launch_bounds__(kThreads, 1)
mx_product_kernel(const __grid_constant__ ProductArgs args,
                  const __grid_constant__ MapsOf<FEW> maps) {
    ProductArgs a = args;
    extern __shared__ char smem_raw[];
    // swizzle atoms repeat every 1024 bytes of shared memory
    const uint32_t raw = saddr(smem_raw);
    const uint32_t smem = (raw + 1023u) & ~1023u;
    const int U = a.units, cap = a.cap;
    // Scale buffers in use. No more than units in flight: a mover that waits for
    // the buffer of unit g - B knows that unit's products are done, and so that
    // `ready` of unit g - U counts no more when it arrives there for unit g.
    const int B = min(kScales, U);
    const uint32_t stage = (uint32_t)stage_bytes(cap, a.outs);
    const uint32_t slots = smem + 2 * U * stage, slot = (uint32_t)slot_bytes(cap, a.outs);
    char *bars = smem_raw + (smem - raw) + 2 * U * stage + kScales * slot;
    // ready: a unit's codes are in shared memory and its scales in tensor memory
    uint64_t *ready = reinterpret_cast<uint64_t *>(bars);
    uint64_t *empty = ready + kMaxUnits;  // per stage
    uint64_t *sfull = empty + 2 * kMaxUnits, *sempty = sfull + kScales;
    uint64_t *sfree = sempty + kScales;   // per scale buffer in tensor memory
    uint64_t *dfull = sfree + kScales, *dempty = dfull + 2, *drain = dempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<int *>(tmem_slot + 1);
    int *tile_count = reinterpret_cast<int *>(tmem_slot + 2);
    int *no_join = reinterpret_cast<int *>(tmem_slot + 3);
    int4 *few_tiles = reinterpret_cast<int4 *>(bars + kBarBytes);
    int32_t *few_pairs = reinterpret_cast<int32_t *>(few_tiles + kFewPairs);
    int32_t *few_rows = few_pairs + kFewPairs * kFewCap;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < U; ++i) {
            bar_init(&ready[i], !FEW ? 5 : a.spread ? 9 : 6);
            bar_init(&empty[2 * i], 1);
            bar_init(&empty[2 * i + 1], 1);
        }
        for (int i = 0; i < kScales; ++i) {
            bar_init(&sfull[i], !FEW ? 1 : a.spread ? 5 : 2);
            bar_init(&sempty[i], 4);
            bar_init(&sfree[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&dfull[i], 1);
            bar_init(&dempty[i], FEW ? 4 : 8);
        }
        bar_init(drain, 1);
        *abort_flag = 0;
        bar_fence_init();
    }
    if (warp == kProducer && lane == 1) {
        prefetch_map(&maps.w);
        prefetch_map(&maps.ws);
    }
    if (warp == kTmemWarp) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
        tc_fence_before();
    }
    grid_dep_wait();
    grid_dep_launch();
    // The state of few rows outlives the call. One whose wait ran out leaves its
    // error word set and counts parts that never came: until the caller has
    // cleared both, its calls share no item.
    if (FEW && threadIdx.x == 0)
        *no_join = a.width > kSaved * kUnit ? *(volatile int32_t *)(a.hdr + 3) : 0;
    if (FEW && a.sel) {
        if (warp == kScaleWarp) {
            bool bad;
            const int n = sort_few(a, lane, few_tiles, few_pairs, few_rows, bad);
            if (lane == 0) {
                *tile_count = n;
                if (blockIdx.x == 0) a.hdr[0] = bad ? IQK_DEVERR_EXPERT : 0;
            }
        }
        a.tiles = few_tiles;
        a.order = few_pairs;
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: two accumulators of `cap`, then the scale buffers, 16 columns
    // a side and buffer (four words a row group, 128 rows)
    const uint32_t scale_col = tmem + 2 * cap;
    const Plan plan = make_plan(a, !a.tiles ? 0 : FEW ? *tile_count : a.hdr[1],
                                !FEW || *no_join == 0);

    auto give_up = [&]() {
        if (!*abort_flag) {
            *abort_flag = 1;
            atomicOr(a.hdr + 3, IQK_DEVERR_TIMEOUT);
            atomicOr(&device_errors, IQK_DEVERR_TIMEOUT);
        }
    };
    const uint32_t off_b = (uint32_t)a.outs * 128, off_sb = (uint32_t)a.outs * 16;
    const int width = (int)a.width, item_stages = (width + kStageK - 1) / kStageK;

    if (warp == kProducer) {
        if (lane == 0) {
            int g = 0;
            Ring ring;
            bool ok = true;
            Part q;
            for (uint32_t i = 0; ok && !*abort_flag && part_of(plan, i, q); ++i) {
                int out0;
                const int4 tl = tile_of(a, plan, q.item, out0);
                const int box = box_of(a, tl);
                // few rows: written by the rounding warps
                const uint32_t bytes = (uint32_t)(128 * (a.outs + (FEW ? 0 : 16 << box)));
                const int row0 = (int)((int64_t)tl.x * a.out_features + out0);
                for (int u = q.u0; ok && u < q.u1; ++u, ++g, ring.next(U)) {
                    // the last unit's second half may lie past the width
                    const int halves = min(2, item_stages - 2 * u);
                    for (int h = 0; h < halves; ++h) {
                        const int s = 2 * ring.s + h;
                        if (!bar_wait_poll(&empty[s], ring.phase ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        if (h == 0) bar_expect_tx(&ready[ring.s], halves * bytes);
                        const uint32_t st = smem + s * stage;
                        tma_2d(st, &maps.w, u * 256 + h * 128, row0, &ready[ring.s]);
                        if constexpr (!FEW)
                            tma_2d(st + off_b, &maps.x[box], u * 256 + h * 128, tl.y, &ready[ring.s]);
                    }
                }
            }
            if (!ok) give_up();
            for (int d = 0; d < U && d < g; ++d) {  // every copy lands before the CTA exits
                const int gg = g - 1 - d;
                if (!bar_wait_poll(&ready[gg % U], (uint32_t)(gg / U) & 1u, nullptr)) give_up();
            }
        }
        __syncwarp();
    } else if (warp == kScaleWarp) {
        if (lane == 0) {
            int g = 0;
            Ring ring;
            bool ok = true;
            Part q;
            for (uint32_t i = 0; ok && !*abort_flag && part_of(plan, i, q); ++i) {
                int out0;
                const int4 tl = tile_of(a, plan, q.item, out0);
                const int box = box_of(a, tl);
                const uint32_t bytes = (uint32_t)(16 * (a.outs + (FEW ? 0 : 16 << box)));
                const int row0 = (int)((int64_t)tl.x * a.out_features + out0);
                for (int u = q.u0; u < q.u1; ++u, ++g, ring.next(B)) {
                    const int b = ring.s;
                    if (!bar_wait_poll(&sempty[b], ring.phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    bar_expect_tx(&sfull[b], bytes);
                    tma_2d(slots + b * slot, &maps.ws, u * 16, row0, &sfull[b]);
                    if constexpr (!FEW)
                        tma_2d(slots + b * slot + off_sb, &maps.xs[box], u * 16, tl.y, &sfull[b]);
                }
            }
            if (!ok) give_up();
            for (int d = 0; d < B && d < g; ++d) {
                const int gg = g - 1 - d;
                if (!bar_wait_poll(&sfull[gg % B], (uint32_t)(gg / B) & 1u, nullptr)) give_up();
            }
        }
        __syncwarp();
    } else if (warp == kIssuer) {
        // One warp's dependent instructions bound this loop, so it is bare: the
        // issuing lane is elected once, one barrier says that a unit's codes and
        // scales are there, and a product's operands are adds to the unit's.
        const bool leader = elect_one();
        const int last_steps = (width - (item_stages - 1) * kStageK + 63) / 64;
        const uint64_t desc0 = sw128_desc(smem);
        const uint32_t desc_stage = stage >> 4, desc_b = off_b >> 4;
        int n = 0, b = 0;  // b: the unit's scale buffer
        Ring ring;
        bool ok = true;
        Part q;
        for (uint32_t i = 0; ok && part_of(plan, i, q); ++i, ++n) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int npad = (tl.z + 15) & ~15;
            const uint32_t even = idesc_mxf4(kOuts, npad, 0), odd = idesc_mxf4(kOuts, npad, 2);
            const int acc = n & 1;
            const uint32_t d = tmem + acc * cap;
            if (n >= 2)
                ok = bar_wait_poll(&dempty[acc], ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag);
            for (int u = q.u0; u < q.u1; ++u, ring.next(U), b = b + 1 == B ? 0 : b + 1) {
                const int left = item_stages - 2 * u;  // stages from here
                ok = ok && bar_wait_poll(&ready[ring.s], ring.phase, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    // a step is 32 bytes of each operand: 2 in a descriptor's 16-byte units
                    const uint64_t da = desc0 + 2 * ring.s * desc_stage, db = da + desc_b;
                    const uint64_t ea = da + desc_stage, eb = ea + desc_b;
                    const uint32_t sa = scale_col + b * 32, sb = sa + 16;
                    const uint32_t more = u > q.u0 ? 1u : 0u;
                    if (left > 2 || (left == 2 && last_steps == 4)) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc_mma_mxf4(d, da + 2 * k, db + 2 * k, k & 1 ? odd : even,
                                        sa + (k >> 1) * 4, sb + (k >> 1) * 4, k ? 1u : more);
                        tc_commit(&empty[2 * ring.s]);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc_mma_mxf4(d, ea + 2 * k, eb + 2 * k, k & 1 ? odd : even,
                                        sa + 8 + (k >> 1) * 4, sb + 8 + (k >> 1) * 4, 1u);
                    } else {
                        const int steps = (left - 1) * 4 + last_steps;
                        for (int k = 0; k < steps; ++k) {
                            const uint64_t ka = k < 4 ? da + 2 * k : ea + 2 * (k - 4);
                            tc_mma_mxf4(d, ka, ka + desc_b, k & 1 ? odd : even,
                                        sa + (k >> 1) * 4, sb + (k >> 1) * 4, k ? 1u : more);
                        }
                        tc_commit(&empty[2 * ring.s]);
                    }
                    tc_commit(&empty[2 * ring.s + 1]);  // in any case: its phase counts units
                    tc_commit(&sfree[b]);
                    if (u + 1 == q.u1) tc_commit(&dfull[acc]);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && lane == 0) give_up();
        __syncwarp();
        if (leader) tc_commit(drain);  // every MMA ends before tensor memory is freed
        __syncwarp();
    } else if (warp >= kMover0 && warp < kMover0 + 4) {
        const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16;
        Ring ring, buffer;
        bool ok = true;
        Part q;
        for (uint32_t i = 0; ok && part_of(plan, i, q); ++i) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int rows = 16 << box_of(a, tl);
            for (int u = q.u0; u < q.u1; ++u, ring.next(U), buffer.next(B)) {
                const int b = buffer.s;
                ok = bar_wait_poll(&sfull[b], buffer.phase, abort_flag) &&
                     bar_wait_poll(&sfree[b], buffer.phase ^ 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sl = slots + b * slot;
                const uint32_t dst = scale_col + quarter + b * 32;
                uint4 w[4], x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 32 * j + lane;
                    w[j] = r < a.outs ? lds128(sl + r * 16) : make_uint4(0u, 0u, 0u, 0u);
                    x[j] = r < rows ? lds128(sl + off_sb + r * 16) : make_uint4(0u, 0u, 0u, 0u);
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
                if (lane == 0) {
                    bar_arrive(&ready[ring.s]);
                    bar_arrive(&sempty[b]);
                }
            }
        }
        if (!ok) give_up();
    } else if (FEW && warp >= kRound0) {
        // lane: the 32 columns lane % 16 of every other row of this warp's
        const int block = lane & 15, turn = warp - kRound0;
        const int first = (lane >> 4) + (a.spread ? 2 * turn : 0), step = a.spread ? 8 : 2;
        int g = 0;
        Ring ring, scales;
        bool ok = true;
        Part q;
        for (uint32_t i = 0; ok && part_of(plan, i, q); ++i) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            for (int u = q.u0; u < q.u1; ++u, ++g) {
                const int halves = min(2, item_stages - 2 * u);
                const Ring at = ring, buffer = scales;
                ring.next(U);
                scales.next(B);
                if (!a.spread && (g & 3) != turn) continue;
                const int b = buffer.s;
                ok = bar_wait_poll(&empty[2 * at.s], at.phase ^ 1u, abort_flag) &&
                     (halves == 1 ||
                      bar_wait_poll(&empty[2 * at.s + 1], at.phase ^ 1u, abort_flag)) &&
                     bar_wait_poll(&sempty[b], buffer.phase ^ 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t st = smem + (2 * at.s + (block >> 3)) * stage + off_b;
                const uint32_t sl = slots + b * slot + off_sb;
                const int64_t col = (int64_t)u * kUnit + block * kMxBlock;
#pragma unroll 2
                for (int r = first; r < tl.z; r += step) {
                    uint32_t w[4] = {0u, 0u, 0u, 0u}, byte = 0u;
                    if (col < a.width) {
                        const int64_t row = a.tiles ? few_rows[tl.y + r] : tl.y + r;
                        const XT *src = static_cast<const XT *>(a.x) + row * a.x_stride + col;
                        float v[4][8];
                        uint32_t amax = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (a.wide) load8<XT, true>(src + 8 * j, v[j]);
                            else load8<XT, false>(src + 8 * j, v[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            amax = max(amax, __float_as_uint(v[j >> 3][j & 7]) & 0x7fffffffu);
                        float inv;
                        byte = scale_byte(amax, inv);
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = codes8(v[j], inv);
                    }
                    // row r of the swizzle atom of 256 columns, its 16-byte chunk block % 8;
                    // the scale byte in any case, codes where the unit has the half
                    const uint32_t to = st + r * 128 + ((uint32_t)((block & 7) ^ (r & 7)) << 4);
                    if (block < 8 || halves == 2)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(to),
                                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    asm volatile("st.shared.u8 [%0], %1;\n" ::"r"(sl + r * 16 + block),
                                 "r"(byte)
                                 : "memory");
                }
                // the MMA reads shared memory through the asynchronous proxy
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    bar_arrive(&ready[at.s]);
                    bar_arrive(&sfull[b]);
                }
            }
        }
        if (!ok) give_up();
    } else if (warp >= kEpi0) {
        const int quarter = warp & 3;
        const int r = 32 * quarter + lane;  // this thread's output of the item
        const bool active = 32 * quarter < a.outs;
        const int half = (warp - kEpi0) / 4;
        const bool pairs = a.out_features % 2 == 0 && reinterpret_cast<uintptr_t>(a.y) % 4 == 0;
        int n = 0;
        Part q;
        for (uint32_t i = 0; part_of(plan, i, q); ++i, ++n) {
            int out0;
            const int4 tl = tile_of(a, plan, q.item, out0);
            const int acc = n & 1;
            const bool ok = bar_wait_poll(&dfull[acc], (uint32_t)(n >> 1) & 1u, abort_flag);
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
            // this warp's rows of the tile
            const int cut = FEW ? tl.z : min(tl.z, ((tl.z + 1) / 2 + 15) & ~15);
            const int c0 = half ? cut : 0, c1 = half ? tl.z : cut;
            for (int c = c0; active && c < c1; c += 16) {
                uint32_t d[2][8];
                const int here = min(16, c1 - c);
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
            if (whole || !active) continue;
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
            if (lane == 0) done = (uint32_t)atomicAdd(&a.tickets[shared_item * 8 + half * 4 + quarter], 1);
            if (__shfl_sync(0xffffffffu, done, 0) != o1 - o0) continue;
            __threadfence();
            // no part is left to count: the ticket is 0 again for the next call
            if (lane == 0) a.tickets[shared_item * 8 + half * 4 + quarter] = 0;
            // the first owner's run may have begun in an earlier item
            const bool early = plan.start(o0) / plan.units != shared_item;
            constexpr int kBatch = 16;  // loads under way
            for (int c = c0; c < c1; c += kBatch) {
                float v[kBatch] = {};
                const int here = min(kBatch, c1 - c);
                for (uint32_t o = o0; o <= o1; ++o) {
                    const float *part = a.slots +
                        ((int64_t)o * 2 + (o == o0 && early ? 1 : 0)) * cap * kOuts + c * kOuts + r;
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (j < here) v[j] += __ldcg(part + j * kOuts);
                }
                store_columns<kBatch>(a, v, here, row_base(a, tl, c, lane), lane, out0 + r, pairs);
            }
        }
    }
    if (warp == kTmemWarp) {  // rows of pairs without an expert
        const int64_t at = blockIdx.x, step = gridDim.x;
        if (FEW && a.sel) {
            for (int64_t p = at; p < a.pairs; p += step)
                if (a.sel[p] < 0 || a.sel[p] >= a.experts) zero_row(a, p, lane);
        } else if (a.tiles) {
            for (int64_t i = a.hdr[2] + at; i < a.pairs; i += step) zero_row(a, a.order[i], lane);
        }
    }
    __syncthreads();
    if (warp == kTmemWarp) {
        if (lane == 0 && !bar_wait_poll(drain, 0, nullptr)) give_up();
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

namespace {

// The shape of an item: `cap` rows, `outs` outputs. A round of items costs a
// CTA, per unit, the bytes that it loads (512 columns of rows and outputs, 272
// bytes each) at its share of the memory's 6500 bytes a ns, or at the 90 that
// one SM can take, and 0.3 us at least for the steps from a load to the next.
// Large items load least in all; small ones fill the SMs. A smaller shape is
// taken where it saves a tenth or more.
struct Shape {
    int cap, outs;
};

Shape shape_of(int64_t pairs, int64_t experts, int64_t out_features, int most) {
    const int64_t used = experts < pairs ? experts : pairs;
    const int64_t mean = (pairs + used - 1) / used;  // rows of an expert
    Shape best{0, 0};
    double least = 0;
    for (int cap = most; cap >= 16; cap /= 2) {
        // an expert's rows vary: below twice the mean many experts would take a
        // second tile, above it the tile's rows (and its stages) are wasted
        if (cap > 16 && cap / 2 >= 2 * mean) continue;
        const int64_t tiles = experts == 1 ? (pairs + cap - 1) / cap
                                           : used + (pairs - used) / cap;
        const int64_t rows = mean < cap ? mean : cap;
        for (int outs = kOuts; outs >= 32; outs /= 2) {
            const int64_t items = tiles * ((out_features + outs - 1) / outs);
            const double bytes = 272.0 * (double)(rows + outs);
            auto round = [&](int64_t ctas) {
                const double shared = bytes * (double)ctas / 6500.0, alone = bytes / 90.0;
                const double ns = shared > alone ? shared : alone;
                return ns > 300.0 ? ns : 300.0;
            };
            const int64_t rest = items % kMaxCtas;
            const double cost = (double)(items / kMaxCtas) * round(kMaxCtas) +
                                (rest ? round(rest) : 0.0);
            if (!best.cap || cost < 0.9 * least) {
                best = Shape{cap, outs};
                least = cost;
            }
        }
    }
    return best;
}

}  // namespace

// A round's share of an item is a unit at least, so what sharing saves is below
// the item's units (make_plan).
bool mx_may_join(int64_t width) { return width > (int64_t)kSaved * kUnit; }

MxLayout mx_layout(int64_t pairs, int64_t num_experts, int64_t width, int64_t out_features) {
    MxLayout L{};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += (bytes + 255) & ~size_t(255);
        return at;
    };
    // a call of no pairs has the shape of a call of one
    const Shape shape = shape_of(pairs > 0 ? pairs : 1, num_experts, out_features, 128);
    L.cap = shape.cap;
    L.outs = shape.outs;
    L.pitch = (width / kMxBlock + 15) / 16 * 16;
    L.max_tiles = (num_experts < pairs ? num_experts : pairs) + pairs / L.cap + 1;
    L.hdr = take(64);
    L.tickets = take(sizeof(int32_t) * 8 * kMaxCtas);
    L.order = take(sizeof(int32_t) * (size_t)pairs);
    L.place = take(sizeof(int32_t) * (size_t)((pairs + 3) / 4 * 4));
    L.tiles = take(16 * (size_t)L.max_tiles);
    L.codes = take((size_t)pairs * (size_t)(width / 2));
    L.scales = take((size_t)pairs * (size_t)L.pitch);
    L.slots = take(mx_may_join(width) ? sizeof(float) * 2 * kMaxCtas * kOuts * (size_t)L.cap : 0);
    L.total = off;
    return L;
}

namespace {

template <bool FEW, typename XT>
cudaError_t launch_kernel(const ProductArgs &a, const MapsOf<FEW> &maps, int sms,
                          cudaStream_t stream) {
    static std::atomic<bool> attr_done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
    if (dev < 0 || !attr_done[dev].load()) {
        const cudaError_t err = cudaFuncSetAttribute(
            mx_product_kernel<FEW, XT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap);
        if (err != cudaSuccess) return err;
        if (dev >= 0) attr_done[dev].store(true);
    }
    const int smem = smem_fixed(a.cap, a.outs) + 2 * a.units * stage_bytes(a.cap, a.outs);
    const int grid = sms < kMaxCtas ? sms : kMaxCtas;
    PdlLaunch pl((unsigned)grid, kThreads, (size_t)smem, stream);
    return cudaLaunchKernelEx(&pl.cfg, mx_product_kernel<FEW, XT>, a, maps);
}

cudaError_t encode_matrix(MatrixMaps &maps, const uint8_t *codes, const uint8_t *scales,
                          int64_t scale_stride, int64_t rows, int64_t width, int outs) {
    const uint64_t code_row = (uint64_t)width / 2, scale_row = (uint64_t)width / kMxBlock;
    const cudaError_t err =
        encode_rows(&maps.w, codes, code_row, (uint64_t)rows, code_row, 128, (uint32_t)outs, true);
    if (err != cudaSuccess) return err;
    return encode_rows(&maps.ws, scales, scale_row, (uint64_t)rows, (uint64_t)scale_stride, 16,
                       (uint32_t)outs, false);
}

}  // namespace

cudaError_t launch_mx_product(const MxProduct &p, cudaStream_t stream, int sms) {
    ProductArgs a{};
    a.out_features = p.out_features;
    a.width = p.width;
    a.pairs = p.pairs;
    a.cap = p.L.cap;
    a.outs = p.L.outs;
    a.units = units_for(a.cap, a.outs);
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
    cudaError_t err = encode_matrix(maps, p.codes, p.scales, p.scale_stride,
                                    p.num_experts * p.out_features, p.width, a.outs);
    const uint64_t code_row = (uint64_t)p.width / 2, scale_row = (uint64_t)p.width / kMxBlock;
    for (int i = 0; i < kBoxes && err == cudaSuccess && (16 << i) <= a.cap; ++i) {
        if (!p.routed && (16 << i) != a.cap) continue;
        err = encode_rows(&maps.x[i], p.ws + p.L.codes, code_row, (uint64_t)p.pairs, code_row, 128,
                          16u << i, true);
        if (err == cudaSuccess)
            err = encode_rows(&maps.xs[i], p.ws + p.L.scales, scale_row, (uint64_t)p.pairs,
                              (uint64_t)p.L.pitch, 16, 16u << i, false);
    }
    if (err != cudaSuccess) return err;
    return launch_kernel<false, float>(a, maps, sms, stream);
}

cudaError_t mx_error_word(int32_t **word) {
    return cudaGetSymbolAddress(reinterpret_cast<void **>(word), device_errors);
}

// State of the one-launch product: hdr, tickets, slots.
constexpr size_t kStateTickets = 256;
constexpr size_t kStateSlots = kStateTickets + (sizeof(int32_t) * 8 * kMaxCtas + 255) / 256 * 256;

static_assert(kStateSlots <= 8192, "the caller clears 8192 bytes");

size_t mx_few_state_bytes(int64_t width) {
    if (!mx_may_join(width)) return kStateTickets;  // no item is shared
    return kStateSlots + sizeof(float) * 2 * kMaxCtas * kOuts * kFewCap;
}

// One launch serves few rows: each CTA rounds the rows that it needs, and sorts
// the pairs, by itself. A lone matrix of up to 16 rows is read once either way;
// above that (64 at most) its tiles read it again, and this form is taken while
// the call has under four units of work a CTA, where launches cost more.
bool mx_few_fits(int64_t pairs, int64_t num_experts, int64_t out_features, int64_t width,
                 bool routed) {
    if (pairs > kFewPairs) return false;
    if (routed || pairs <= kFewCap) return true;
    const int64_t items = (pairs + kFewCap - 1) / kFewCap * ((out_features + kOuts - 1) / kOuts);
    return items * ((width + kUnit - 1) / kUnit) <= 4 * kMaxCtas;
}

cudaError_t launch_mx_few(const MxFew &p, cudaStream_t stream, int sms) {
    ProductArgs a{};
    a.out_features = p.out_features;
    a.width = p.width;
    a.pairs = p.pairs;
    a.cap = kFewCap;
    a.outs = shape_of(p.pairs, p.num_experts, p.out_features, kFewCap).outs;
    a.units = units_for(a.cap, a.outs);
    a.hdr = reinterpret_cast<int32_t *>(p.state);
    a.tickets = reinterpret_cast<int32_t *>(p.state + kStateTickets);
    a.slots = reinterpret_cast<float *>(p.state + kStateSlots);
    a.y = p.y;
    a.y_dtype = p.y_dtype;
    a.x = p.x;
    a.x_stride = p.x_stride;
    a.sel = p.sel;
    a.per_row = (int)(p.pairs / p.x_rows);
    a.experts = (int)p.num_experts;
    const size_t item = p.x_dtype == IQK_F32 ? 4 : 2;
    a.spread = !p.sel && p.pairs > 4;
    a.wide = aligned(p.x, 16) && p.x_stride * (int64_t)item % 16 == 0;
    MatrixMaps maps;
    const cudaError_t err = encode_matrix(maps, p.codes, p.scales, p.scale_stride,
                                          p.num_experts * p.out_features, p.width, a.outs);
    if (err != cudaSuccess) return err;
    if (p.x_dtype == IQK_F32) return launch_kernel<true, float>(a, maps, sms, stream);
    if (p.x_dtype == IQK_F16) return launch_kernel<true, __half>(a, maps, sms, stream);
    return launch_kernel<true, __nv_bfloat16>(a, maps, sms, stream);
}

}  // namespace iqk
