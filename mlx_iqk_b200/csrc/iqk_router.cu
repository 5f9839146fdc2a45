// Expert router: top-k choice with router weights, per-expert counts and the
// balance loss, and their gradient (sm_100a).
//
// One token's logits z[0..E) are one warp's registers. With u(z) = exp(z) for softmax scoring and the logistic
// function for sigmoid scoring, every quantity of a row is a ratio of
//
//   r_e = u(z_e) / u(c),  c the row's largest logit (softmax) or min(it, 0)
//
// so nothing overflows and the denominators below are at least 1/2:
//
//   s_e = r_e / sum_e r_e               score, normalised over the experts
//   choice: the k largest z (ties: the lowest index); -inf is no expert
//   w_j  = scale * r_{i_j} / sum_j r_{i_j}         renormalised weights
//   w_j  = scale * s_{i_j} | scale * sigmoid(z_{i_j})     otherwise
//   f_ge = E count_ge / (k N_g),  P_ge = (1 / N_g) sum_t s_te
//   loss = mean over segments g with N_g > 0 of sum_e f_ge P_ge
//
// A segment is a run of rows (packed sequences); N_g counts its rows that the
// mask keeps and that have a logit above -inf (or NaN). A row may be in none. Gradients, with h_e = 1 (softmax)
// or 1 - sigmoid(z_e), a_e = dloss f_ge / (N_g G'), q = w / scale and g the
// weights' gradient:
//
//   balance        dz_e   += s_e h_e (a_e - sum s a)
//   renormalised   dz_i_j += scale q_j h (g_j - sum q g)
//   softmax        dz_e   += scale s_e ([e = i_j] g_j - sum_j q_j g_j)
//   sigmoid        dz_i_j += scale q_j (1 - q_j) g_j
//
// Sums over rows are joined in a fixed order: a block writes one record per
// segment that it meets, and the finishing kernel adds the records in an order
// that its launch alone decides, so a result repeats bit for bit.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <type_traits>

#include "iqk_common.cuh"
#include "iqk_host.cuh"

namespace iqk {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;  // lane j keeps choice j
constexpr unsigned kFull = 0xffffffffu;

struct RouteArgs {
    const void *logits;
    int64_t tokens, stride;
    int experts, top_k, sigmoid, renormalize;
    float scale;
    const uint8_t *mask;     // [tokens] or null
    const int32_t *offsets;  // [segments + 1] or null (one segment)
    int segments;
    int32_t *indices;        // [tokens, top_k]
    float *weights;          // [tokens, top_k]
    // records: (block + segment) is a record's place, unique because a block
    // meets segments in order
    float *rec_score;        // [records, experts]
    int32_t *rec_count;      // [records, experts]
    int32_t *rec_rows;       // [records]
    int64_t per_block;       // rows of one block (backward: of one warp)
};

__device__ __forceinline__ float logistic(float z) { return 1.f / (1.f + expf(-z)); }

// u(z) / u(c): see the head of the file.
__device__ __forceinline__ float ratio(float z, float c, int sigmoid) {
    if (!sigmoid) return expf(z - c);
    return z >= 0.f ? 1.f / (1.f + expf(-z)) : expf(z - c) / (1.f + expf(z));
}

template <int V>
__device__ __forceinline__ void ratios(const float (&z)[V], float c, int sigmoid, float (&r)[V]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = ratio(z[i], c, 1);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = expf(z[i] - c);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Order-preserving key of a logit. Adding +0 makes -0 equal to +0 and every NaN
// the one whose key is above all numbers'; -inf (no expert, and places past E)
// is the one value whose key is below kNone.
constexpr uint32_t kNone = 0x00800000u;
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}

// The segment of row t and the row after that segment's end: the largest g
// with offsets[g] <= t. -1 or `segments`: no segment.
__device__ __forceinline__ int segment_of(const int32_t *offsets, int segments, int64_t t,
                                          int64_t &end) {
    if (!offsets) return 0;
    int lo = 0, hi = segments + 1;  // offsets[lo - 1] <= t < offsets[hi]
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    if (lo <= segments && offsets[lo] < end) end = offsets[lo];
    return lo - 1;
}

// Value i of lane l is expert (i / N) 32 N + l N + i % N: N values to a load
// (16 bytes where rows allow it, else one).
template <int N> __device__ __forceinline__ int expert_of(int lane, int i) {
    return (i / N) * 32 * N + lane * N + i % N;
}

// One row; places past E read -inf.
template <typename T, int V, int N>
__device__ __forceinline__ void load_row(const RouteArgs &a, int64_t t, int lane, float (&z)[V]) {
    const T *row = static_cast<const T *>(a.logits) + t * a.stride;
#pragma unroll
    for (int i = 0; i < V; i += N) {
        const int e = expert_of<N>(lane, i);
        if constexpr (N == 1) {
            z[i] = e < a.experts ? to_float<T>(row[e]) : -CUDART_INF_F;
        } else {  // E is a multiple of N
            if (e < a.experts) {
                const uint4 u = *reinterpret_cast<const uint4 *>(row + e);
                const T *v = reinterpret_cast<const T *>(&u);
#pragma unroll
                for (int j = 0; j < N; ++j) z[i + j] = to_float<T>(v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) z[i + j] = -CUDART_INF_F;
            }
        }
    }
}

// The key of the row's largest logit; below kNone where the row has no expert.
template <int V> __device__ __forceinline__ uint32_t row_peak(const float (&z)[V]) {
    float best = z[0];
#pragma unroll
    for (int i = 1; i < V; ++i)  // NaN wins, as in the keys
        asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(best) : "f"(z[i]));
    return __reduce_max_sync(kFull, key_of(best));
}

// Lane j gets choice j of the top_k largest (index -1 past the last).
//
// A 16-bit logit fills the upper 22 bits of its f32 key at most, and 1023 -
// expert the ten below: one warp maximum finds the largest and, among equals,
// the first. With up to eight values a lane, each lane sorts its own first (19
// exchanges); then a choice is the maximum of the lanes' heads, and the lane
// that held it moves up its list: 14 instructions a choice for the 35 of a
// search through unsorted values.
template <typename T, int V, int N> struct Sorted {
    uint32_t key[V];
    __device__ __forceinline__ explicit Sorted(const float (&z)[V], int lane) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            key[i] = (key_of(z[i]) & ~1023u) | (1023u - expert_of<N>(lane, i));
        // odd-even merge sort, falling
#pragma unroll
        for (int p = 1; p < V; p *= 2)
#pragma unroll
            for (int k = p; k >= 1; k /= 2)
#pragma unroll
                for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                    for (int i = 0; i < k; ++i)
                        if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                            const uint32_t a = key[i + j], b = key[i + j + k];
                            key[i + j] = max(a, b);
                            key[i + j + k] = min(a, b);
                        }
    }
    __device__ __forceinline__ uint32_t peak() const { return __reduce_max_sync(kFull, key[0]); }
    // the low bits of a negative value's key are the ones of a zero
    __device__ __forceinline__ static float logit(uint32_t top) {
        return value_of((top & ~1023u) | ((top >> 31) ? 0u : 1023u));
    }
    __device__ __forceinline__ void choose(const RouteArgs &a, int lane, uint32_t top, int &index,
                                           float &value) {
        index = -1;
        value = -CUDART_INF_F;
        for (int j = 0; top >= kNone; top = peak()) {
            if (lane == j) {
                index = 1023 - (int)(top & 1023u);
                value = logit(top);
            }
            if (++j == a.top_k) break;
            if (key[0] == top) {
#pragma unroll
                for (int i = 0; i + 1 < V; ++i) key[i] = key[i + 1];
                key[V - 1] = 0;
            }
        }
    }
};

// Unsorted: 32-bit keys, whose expert takes a second warp maximum, and rows of
// more than eight values a lane, where a sort costs more than it saves.
template <typename T, int V, int N>
__device__ __forceinline__ void choose(const RouteArgs &a, const float (&z)[V], int lane,
                                       int &index, float &value) {
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = key_of(z[i]);
    index = -1;
    value = -CUDART_INF_F;
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) best = max(best, key[i]);
        const uint32_t top = __reduce_max_sync(kFull, best);
        if (top < kNone) break;
        int first = kMaxExperts;
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
            if (key[i] == top) first = expert_of<N>(lane, i);
        first = __reduce_min_sync(kFull, first);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (first == expert_of<N>(lane, i)) key[i] = 0;
        if (lane == j) {
            index = first;
            value = value_of(top);
        }
    }
}

struct Nothing {
    template <typename Z> __device__ __forceinline__ Nothing(const Z &, int) {}
};

template <typename T, int V, int N, bool CHOOSE, bool BALANCE>
__device__ __forceinline__ bool route_row(const RouteArgs &a, int64_t t, int lane,
                                          float (&score)[V], int &index) {
    const int k = a.top_k;
    if (a.mask && !a.mask[t]) {
        if (CHOOSE && lane < k) {
            a.indices[t * k + lane] = -1;
            a.weights[t * k + lane] = 0.f;
        }
        return false;
    }
    float z[V];
    load_row<T, V, N>(a, t, lane, z);
    constexpr bool kSort = CHOOSE && sizeof(T) == 2 && V <= 8;
    typename std::conditional<kSort, Sorted<T, V, N>, Nothing>::type sorted(z, lane);
    uint32_t peak;
    if constexpr (kSort) peak = sorted.peak();
    else peak = row_peak<V>(z);
    const float top = kSort ? Sorted<T, V, N>::logit(peak) : value_of(peak);
    const float c = a.sigmoid ? fminf(top, 0.f) : top;
    float total = 1.f;
    if (BALANCE || (CHOOSE && !a.renormalize && !a.sigmoid)) {
        float part = 0.f;
        ratios<V>(z, c, a.sigmoid, score);
#pragma unroll
        for (int i = 0; i < V; ++i) part += score[i];
        total = warp_sum(part);
    }
    if (CHOOSE) {
        float value, w;
        if constexpr (kSort) sorted.choose(a, lane, peak, index, value);
        else choose<T, V, N>(a, z, lane, index, value);
        if (a.renormalize) {
            const float r = index >= 0 ? ratio(value, c, a.sigmoid) : 0.f;
            w = r / warp_sum(r);
        } else {
            w = a.sigmoid ? logistic(value) : ratio(value, c, 0) / total;
        }
        if (lane < k) {
            a.indices[t * k + lane] = index;
            a.weights[t * k + lane] = index >= 0 ? w * a.scale : 0.f;
        }
    } else {
        index = lane < k ? a.indices[t * k + lane] : -1;
    }
    if (BALANCE) {
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < V; ++i) score[i] *= inv;
    }
    return peak >= kNone;
}

// A warp a row.
template <typename T, int V, int N>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.tokens;
         t += step) {
        float score[V];
        int index;
        route_row<T, V, N, true, false>(a, t, lane, score, index);
    }
}

// A block takes per_block rows in a run; its warps share the rows of each
// segment part, and the part's sums become one record.
// Warps of a balance block: a row's registers and the warps' sums (48 KB of
// shared memory at most) bound them.
__host__ __device__ constexpr int balance_warps(int v) { return v <= 8 ? 32 : v <= 16 ? 16 : 8; }

template <typename T, int V, int N, bool CHOOSE>
__global__ void __launch_bounds__(32 * balance_warps(V)) balance_kernel(RouteArgs a) {
    extern __shared__ float sums[];  // [warps, experts], then the counts
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t *counts = reinterpret_cast<int32_t *>(sums + warps * a.experts);
    __shared__ int rows;
    const int64_t b0 = (int64_t)blockIdx.x * a.per_block;
    const int64_t b1 = min(b0 + a.per_block, a.tokens);
    for (int64_t t0 = b0; t0 < b1;) {
        int64_t t1 = b1;
        const int g = segment_of(a.offsets, a.segments, t0, t1);
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
        for (int e = threadIdx.x; e < a.experts; e += blockDim.x) counts[e] = 0;
        if (threadIdx.x == 0) rows = 0;
        __syncthreads();
        int mine = 0;
        for (int64_t t = t0 + warp; t < t1; t += warps) {
            float score[V];
            int index = -1;
            if (!route_row<T, V, N, CHOOSE, true>(a, t, lane, score, index)) continue;
            ++mine;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += score[i];
            if (lane < a.top_k && index >= 0 && index < a.experts) atomicAdd(&counts[index], 1);
        }
        if (lane == 0) atomicAdd(&rows, mine);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (expert_of<N>(lane, i) < a.experts)
                sums[warp * a.experts + expert_of<N>(lane, i)] = acc[i];
        __syncthreads();
        if (g >= 0 && g < a.segments) {
            const int64_t rec = blockIdx.x + g;
            for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
                float s = 0.f;
                for (int w = 0; w < warps; ++w) s += sums[w * a.experts + e];
                a.rec_score[rec * a.experts + e] = s;
                a.rec_count[rec * a.experts + e] = counts[e];
            }
            if (threadIdx.x == 0) a.rec_rows[rec] = rows;
        }
        __syncthreads();
        t0 = t1;
    }
}

// The blocks [first, last] that hold a part of segment g; false: no row.
__device__ __forceinline__ bool blocks_of(const RouteArgs &a, int g, int &first, int &last) {
    const int64_t lo = a.offsets ? max(a.offsets[g], 0) : 0;
    const int64_t hi = a.offsets ? min((int64_t)a.offsets[g + 1], a.tokens) : a.tokens;
    if (lo >= hi) return false;
    first = (int)(lo / a.per_block);
    last = (int)((hi - 1) / a.per_block);
    return true;
}

constexpr int kFinishCtas = 8, kFinishWarps = 16;

// The rows of segment g that count, summed by a whole warp.
__device__ __forceinline__ int rows_of(const RouteArgs &a, int g, int lane) {
    int first, last, n = 0;
    if (!blocks_of(a, g, first, last)) return 0;
    for (int b = first + lane; b <= last; b += 32) n += a.rec_rows[b + g];
    return __reduce_add_sync(kFull, n);
}

// Counts, mean scores, the loss, and slope_ge = f_ge / (N_g G'). A cluster of
// eight CTAs shares the experts; in a CTA `share` warps split a segment's
// records (all 16 for one segment, one for 16 or more) and lanes are experts.
__global__ void __cluster_dims__(kFinishCtas, 1, 1) __launch_bounds__(32 * kFinishWarps)
balance_finish_kernel(RouteArgs a, float *loss, int32_t *counts, float *slope) {
    __shared__ float scores[kFinishWarps][32], part_sum[kFinishWarps], total;
    __shared__ int32_t picked[kFinishWarps][32];
    constexpr int kKept = 256;
    __shared__ int filled, kept[kKept];  // rows of the first segments
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) filled = 0;
    __syncthreads();
    int mine = 0;
    for (int g = warp; g < a.segments; g += kFinishWarps) {
        const int n = rows_of(a, g, lane);
        if (lane == 0 && g < kKept) kept[g] = n;
        mine += n > 0;
    }
    if (lane == 0 && mine) atomicAdd(&filled, mine);
    __syncthreads();
    const float mean = 1.f / (float)max(filled, 1);
    int share = kFinishWarps;
    while (share > 1 && share * a.segments > kFinishWarps) share >>= 1;
    const int sub = warp % share;
    float part = 0.f;
    for (int g0 = 0; g0 < a.segments; g0 += kFinishWarps / share) {
        const int g = g0 + warp / share;
        int first = 0, last = -1, n = 0;
        if (g < a.segments && blocks_of(a, g, first, last))
            n = g < kKept ? kept[g] : rows_of(a, g, lane);
        const float inv = n > 0 ? 1.f / (float)n : 0.f;
        for (int e0 = blockIdx.x * 32; e0 < a.experts; e0 += kFinishCtas * 32) {
            const int e = e0 + lane;
            float s = 0.f;
            int c = 0;
            if (e < a.experts) {
#pragma unroll 4
                for (int b = first + sub; b <= last; b += share) {
                    s += a.rec_score[(int64_t)(b + g) * a.experts + e];
                    c += a.rec_count[(int64_t)(b + g) * a.experts + e];
                }
            }
            scores[warp][lane] = s;
            picked[warp][lane] = c;
            __syncthreads();
            if (sub == 0 && g < a.segments && e < a.experts) {
                for (int w = 1; w < share; ++w) {
                    s += scores[warp + w][lane];
                    c += picked[warp + w][lane];
                }
                const float f = (float)c * (float)a.experts * inv / (float)a.top_k;
                part += f * s * inv;
                counts[(int64_t)g * a.experts + e] = c;
                slope[(int64_t)g * a.experts + e] = f * inv * mean;
            }
            __syncthreads();
        }
    }
    part = warp_sum(part);
    if (lane == 0) part_sum[warp] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        float v = 0.f;
        for (int w = 0; w < kFinishWarps; ++w) v += part_sum[w];
        total = v * mean;
    }
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float v = 0.f;
        for (int c = 0; c < kFinishCtas; ++c) v += *cluster.map_shared_rank(&total, c);
        *loss = v;
    }
    cluster.sync();  // a CTA's shared memory stays until it is read
}

struct RouteGrad {
    const float *weights;  // gradient of the weights, or null
    const float *slope;    // [segments, experts], or null
    const float *loss;     // the loss's gradient, one value
    void *logits;          // out, [tokens, experts]
};

// A warp takes a run of rows, so that a segment's slopes stay in registers
// until it ends. Shared memory holds a row for what goes by expert: the chosen
// logits and the chosen experts' part of the gradient.
template <typename T, int V, int N>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a, RouteGrad d) {
    extern __shared__ __align__(16) float rows[];  // [warps, 32 V]
    const int lane = threadIdx.x & 31, k = a.top_k;
    float *row = rows + (threadIdx.x >> 5) * 32 * V;
    const int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t0 = w * a.per_block, t1 = min(t0 + a.per_block, a.tokens);
    const float up = d.slope ? *d.loss : 0.f;
    const bool softmax_all = d.weights && !a.renormalize && !a.sigmoid;
    float slope[V];
    int64_t end = t0;  // of the segment in `slope`
    bool there = false;
    for (int64_t t = t0; t < t1; ++t) {
        T *out = static_cast<T *>(d.logits) + t * a.experts;
        // every load of the row, before anything waits for one
        const bool keep = !a.mask || a.mask[t];
        float z[V], dz[V];
        load_row<T, V, N>(a, t, lane, z);
        int index = -1;
        float g = 0.f;
        if (d.weights && lane < k) {
            index = a.indices[t * k + lane];
            g = d.weights[t * k + lane];
        }
        if (d.slope && t >= end) {
            end = a.tokens;
            const int s = segment_of(a.offsets, a.segments, t, end);
            there = s >= 0 && s < a.segments;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = expert_of<N>(lane, i);
                slope[i] = there && e < a.experts ? up * d.slope[(int64_t)s * a.experts + e] : 0.f;
            }
        }
        const uint32_t peak = keep ? row_peak<V>(z) : 0u;
        if (peak < kNone) {  // no expert: nothing depends on this row
#pragma unroll
            for (int i = 0; i < V; ++i) dz[i] = 0.f;
        } else {
            const float top = value_of(peak);
            const float c = a.sigmoid ? fminf(top, 0.f) : top;
            float inv = 1.f;
            if (there || softmax_all) {
                float part = 0.f;
                ratios<V>(z, c, a.sigmoid, dz);
#pragma unroll
                for (int i = 0; i < V; ++i) part += dz[i];
                inv = 1.f / warp_sum(part);
            }
            // the choice's part: lane j adds `own` at its expert, and every
            // expert takes -s_e * shared (softmax that is not renormalised)
            float own = 0.f, shared = 0.f;
            const bool chosen = index >= 0 && index < a.experts;
            if (d.weights) {
#pragma unroll
                for (int i = 0; i < V; ++i) row[expert_of<N>(lane, i)] = z[i];
                __syncwarp();
                const float zi = chosen ? row[index] : -CUDART_INF_F;
                __syncwarp();
                const float r = chosen ? ratio(zi, c, a.sigmoid) : 0.f;
                const float h = a.sigmoid ? logistic(-zi) : 1.f;
                g = chosen ? g * a.scale : 0.f;
                if (a.renormalize) {
                    const float q = r / warp_sum(r);
                    const float dot = warp_sum(q * g);
                    own = chosen ? q * h * (g - dot) : 0.f;
                } else if (a.sigmoid) {
                    own = chosen ? logistic(zi) * h * g : 0.f;
                } else {
                    own = r * inv * g;
                    shared = warp_sum(own);
                }
            }
            float dot = 0.f;
            if (there) {
#pragma unroll
                for (int i = 0; i < V; ++i) dot += dz[i] * slope[i];
                dot = warp_sum(dot) * inv;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float s = dz[i] * inv;
                const float v = there ? s * (slope[i] - dot) : 0.f;
                dz[i] = softmax_all ? v - s * shared : v;
            }
            if (a.sigmoid && there) {
#pragma unroll
                for (int i = 0; i < V; ++i) dz[i] *= logistic(-z[i]);
            }
            if (d.weights) {
#pragma unroll
                for (int i = 0; i < V; ++i) row[expert_of<N>(lane, i)] = dz[i];
                __syncwarp();
                if (chosen) row[index] += own;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < V; ++i) dz[i] = row[expert_of<N>(lane, i)];
                __syncwarp();
            }
        }
#pragma unroll
        for (int i = 0; i < V; i += N) {
            const int e = expert_of<N>(lane, i);
            if (e >= a.experts) continue;
            if constexpr (N == 1) {
                out[e] = from_float<T>(dz[i]);
            } else {
                uint4 u;
                T *v = reinterpret_cast<T *>(&u);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = from_float<T>(dz[i + j]);
                *reinterpret_cast<uint4 *>(out + e) = u;
            }
        }
    }
}

// 64-bit expert indices to 32 bits: what lies beyond them is held at the type's
// ends, which are no experts. Dropping the upper half would make 2^32 + 3 expert 3.
__global__ void __launch_bounds__(256)
narrow_indices_kernel(const int64_t *__restrict__ in, int64_t count, int32_t *__restrict__ out) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += step)
        out[i] = (int32_t)max((int64_t)INT32_MIN, min((int64_t)INT32_MAX, in[i]));
}

struct RouteLayout {
    size_t score, count, rows, total;
    int64_t blocks, per_block;
};

// Blocks of the balance kernel: one per SM, 32 rows (one a warp) or more each.
RouteLayout route_layout(int64_t tokens, int64_t experts, int64_t segments) {
    RouteLayout L{};
    L.per_block = (tokens + 147) / 148;
    if (L.per_block < 32) L.per_block = 32;
    L.blocks = (tokens + L.per_block - 1) / L.per_block;
    const int64_t records = L.blocks + segments;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += (bytes + 255) & ~size_t(255);
        return at;
    };
    L.score = take(sizeof(float) * (size_t)(records * experts));
    L.count = take(sizeof(int32_t) * (size_t)(records * experts));
    L.rows = take(sizeof(int32_t) * (size_t)records);
    L.total = off;
    return L;
}

template <typename T, int V, int N>
cudaError_t launch_choice(const RouteArgs &a, int sms, cudaStream_t s) {
    const int64_t want = (a.tokens + 7) / 8;
    const int64_t most = (int64_t)sms * 8;
    route_kernel<T, V, N><<<(unsigned)(want < most ? want : most), 256, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V, int N>
cudaError_t launch_balance(const RouteArgs &a, bool choose, int64_t blocks, cudaStream_t s) {
    constexpr int warps = balance_warps(V);
    static_assert((warps + 1) * 32 * V * 4 <= 48 * 1024, "the warps' sums fit shared memory");
    const size_t smem = (size_t)(warps + 1) * a.experts * 4;
    if (choose) balance_kernel<T, V, N, true><<<(unsigned)blocks, 32 * warps, smem, s>>>(a);
    else balance_kernel<T, V, N, false><<<(unsigned)blocks, 32 * warps, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V, int N>
cudaError_t launch_backward(RouteArgs a, const RouteGrad &d, int sms, cudaStream_t s) {
    // rows of a warp: one while that fills the SMs once (32 warps each)
    const int64_t warps = (int64_t)sms * 32;
    a.per_block = (a.tokens + warps - 1) / warps;
    const int64_t used = (a.tokens + a.per_block - 1) / a.per_block;
    route_backward_kernel<T, V, N>
        <<<(unsigned)((used + 7) / 8), 256, (size_t)8 * 32 * V * 4, s>>>(a, d);
    return cudaGetLastError();
}

// Rows may be read and written 16 bytes at a time.
template <typename T> bool wide(const RouteArgs &a, const void *out) {
    const int n = 16 / (int)sizeof(T);
    return a.experts % n == 0 && a.stride * (int64_t)sizeof(T) % 16 == 0 &&
           aligned(a.logits, 16) && aligned(out, 16);
}

// F(T, V, N): V values a lane cover E experts, N to a load.
#define IQK_ROUTE_V(T, W, F)                                             \
    (a.experts <= 64    ? F(T, 2, 1)                                      \
     : a.experts <= 128 ? ((W) && sizeof(T) == 4 ? F(T, 4, 4) : F(T, 4, 1)) \
     : a.experts <= 256 ? ((W) ? F(T, 8, (16 / sizeof(T))) : F(T, 8, 1))  \
     : a.experts <= 512 ? ((W) ? F(T, 16, (16 / sizeof(T))) : F(T, 16, 1)) \
                        : ((W) ? F(T, 32, (16 / sizeof(T))) : F(T, 32, 1)))
#define IQK_ROUTE_TV(dtype, out, F)                                          \
    ((dtype) == IQK_F32   ? IQK_ROUTE_V(float, wide<float>(a, out), F)       \
     : (dtype) == IQK_F16 ? IQK_ROUTE_V(__half, wide<__half>(a, out), F)     \
                          : IQK_ROUTE_V(__nv_bfloat16, wide<__nv_bfloat16>(a, out), F))

size_t element(int dtype) { return dtype == IQK_F32 ? 4 : 2; }

int check_route(const void *logits, int dtype, int64_t tokens, int64_t experts, int64_t stride,
                int top_k, int scoring) {
    if (!dtype_ok(dtype)) return IQK_ERR_ARGUMENT;
    if (scoring != IQK_SOFTMAX && scoring != IQK_SIGMOID) return IQK_ERR_ARGUMENT;
    if (experts <= 0 || experts > kMaxExperts) return IQK_ERR_GEOMETRY;
    if (top_k <= 0 || top_k > kMaxTopK || top_k > experts) return IQK_ERR_GEOMETRY;
    if (tokens < 0 || tokens > ((int64_t)1 << 31) - 1) return IQK_ERR_GEOMETRY;
    if (stride < experts && tokens > 1) return IQK_ERR_GEOMETRY;
    if (tokens == 0) return IQK_OK;
    if (!logits) return IQK_ERR_ARGUMENT;
    if (!aligned(logits, element(dtype))) return IQK_ERR_ALIGNMENT;
    return IQK_OK;
}

RouteArgs route_args(const void *logits, int64_t tokens, int64_t experts, int64_t stride,
                     const uint8_t *mask, int top_k, int scoring) {
    RouteArgs a{};
    a.logits = logits;
    a.tokens = tokens;
    a.stride = stride;
    a.experts = (int)experts;
    a.top_k = top_k;
    a.sigmoid = scoring == IQK_SIGMOID;
    a.mask = mask;
    a.segments = 1;
    return a;
}

}  // namespace
}  // namespace iqk

using namespace iqk;

extern "C" {

int iqk_narrow_indices(const int64_t *indices, int64_t count, int32_t *out, iqk_stream_t stream) {
    if (count < 0) return IQK_ERR_GEOMETRY;
    if (count == 0) return IQK_OK;
    if (!indices || !out) return IQK_ERR_ARGUMENT;
    if (!aligned(indices, 8) || !aligned(out, 4)) return IQK_ERR_ALIGNMENT;
    const int64_t want = (count + 255) / 256, most = (int64_t)num_sms_current() * 8;
    narrow_indices_kernel<<<(unsigned)(want < most ? want : most), 256, 0,
                            reinterpret_cast<cudaStream_t>(stream)>>>(indices, count, out);
    return cuda_status(cudaGetLastError());
}

int iqk_route(const void *logits, int dtype, int64_t tokens, int64_t num_experts,
              int64_t row_stride, const uint8_t *mask, int top_k, int scoring, int renormalize,
              float scale, int32_t *indices, float *weights, iqk_stream_t stream) {
    const int st = check_route(logits, dtype, tokens, num_experts, row_stride, top_k, scoring);
    if (st != IQK_OK || tokens == 0) return st;
    if (!indices || !weights) return IQK_ERR_ARGUMENT;
    if (!aligned(indices, 4) || !aligned(weights, 4)) return IQK_ERR_ALIGNMENT;
    RouteArgs a = route_args(logits, tokens, num_experts, row_stride, mask, top_k, scoring);
    a.renormalize = renormalize != 0;
    a.scale = scale;
    a.indices = indices;
    a.weights = weights;
    const int sms = num_sms_current();
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define IQK_F(T, V, N) launch_choice<T, V, N>(a, sms, s)
    return cuda_status(IQK_ROUTE_TV(dtype, nullptr, IQK_F));
#undef IQK_F
}

size_t iqk_balance_workspace_bytes(int64_t tokens, int64_t num_experts, int64_t segments) {
    if (tokens < 0 || num_experts <= 0 || num_experts > kMaxExperts || segments <= 0) return 0;
    return route_layout(tokens, num_experts, segments).total;
}

int iqk_route_balanced(const void *logits, int dtype, int64_t tokens, int64_t num_experts,
                       int64_t row_stride, const uint8_t *mask, const int32_t *offsets,
                       int64_t segments, int top_k, int scoring, int renormalize, float scale,
                       int32_t *indices, float *weights, float *loss, int32_t *counts,
                       float *slope, void *workspace, size_t workspace_bytes,
                       iqk_stream_t stream) {
    const int st = check_route(logits, dtype, tokens, num_experts, row_stride, top_k, scoring);
    if (st != IQK_OK) return st;
    if (segments <= 0 || segments > (1 << 20) || (!offsets && segments != 1))
        return IQK_ERR_GEOMETRY;
    if (!loss || !counts || !slope || !workspace || (tokens && !indices)) return IQK_ERR_ARGUMENT;
    if (!aligned(indices, 4) || !aligned(weights, 4) || !aligned(loss, 4) ||
        !aligned(counts, 4) || !aligned(slope, 4) || !aligned(offsets, 4) ||
        !aligned(workspace, 256))
        return IQK_ERR_ALIGNMENT;
    const RouteLayout L = route_layout(tokens, num_experts, segments);
    if (workspace_bytes < L.total) return IQK_ERR_WORKSPACE;
    RouteArgs a = route_args(logits, tokens, num_experts, row_stride, mask, top_k, scoring);
    a.renormalize = renormalize != 0;
    a.scale = scale;
    a.offsets = offsets;
    a.segments = (int)segments;
    a.indices = indices;
    a.weights = weights;
    a.per_block = L.per_block;
    char *w = static_cast<char *>(workspace);
    a.rec_score = reinterpret_cast<float *>(w + L.score);
    a.rec_count = reinterpret_cast<int32_t *>(w + L.count);
    a.rec_rows = reinterpret_cast<int32_t *>(w + L.rows);
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t err = cudaSuccess;
#define IQK_F(T, V, N) launch_balance<T, V, N>(a, weights != nullptr, L.blocks, s)
    if (tokens) err = IQK_ROUTE_TV(dtype, nullptr, IQK_F);
#undef IQK_F
    if (err != cudaSuccess) return cuda_status(err);
    balance_finish_kernel<<<kFinishCtas, 32 * kFinishWarps, 0, s>>>(a, loss, counts, slope);
    return cuda_status(cudaGetLastError());
}

int iqk_route_backward(const void *logits, int dtype, int64_t tokens, int64_t num_experts,
                       int64_t row_stride, const uint8_t *mask, const int32_t *offsets,
                       int64_t segments, int top_k, int scoring, int renormalize, float scale,
                       const int32_t *indices, const float *grad_weights, const float *slope,
                       const float *grad_loss, void *grad_logits, iqk_stream_t stream) {
    const int st = check_route(logits, dtype, tokens, num_experts, row_stride, top_k, scoring);
    if (st != IQK_OK || tokens == 0) return st;
    if (segments <= 0 || segments > (1 << 20) || (!offsets && segments != 1))
        return IQK_ERR_GEOMETRY;
    if (!grad_logits || (grad_weights && !indices) || (slope && !grad_loss))
        return IQK_ERR_ARGUMENT;
    if (!aligned(indices, 4) || !aligned(grad_weights, 4) || !aligned(slope, 4) ||
        !aligned(grad_loss, 4) || !aligned(offsets, 4) || !aligned(grad_logits, element(dtype)))
        return IQK_ERR_ALIGNMENT;
    RouteArgs a = route_args(logits, tokens, num_experts, row_stride, mask, top_k, scoring);
    a.renormalize = renormalize != 0;
    a.scale = scale;
    a.offsets = offsets;
    a.segments = (int)segments;
    a.indices = const_cast<int32_t *>(indices);
    const RouteGrad d{grad_weights, slope, grad_loss, grad_logits};
    const int sms = num_sms_current();
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define IQK_F(T, V, N) launch_backward<T, V, N>(a, d, sms, s)
    return cuda_status(IQK_ROUTE_TV(dtype, grad_logits, IQK_F));
#undef IQK_F
}

}  // extern "C"
