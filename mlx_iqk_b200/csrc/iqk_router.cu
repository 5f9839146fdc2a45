// Expert router: top-k choice with router weights, per-expert counts and the
// balance loss, and their gradient (sm_100a).
//
// One token's logits z[0..E) are one warp's registers (lane l holds experts
// l, l + 32, ...). With u(z) = exp(z) for softmax scoring and the logistic
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
// mask keeps and that have a finite logit. Gradients, with h_e = 1 (softmax)
// or 1 - sigmoid(z_e), a_e = dloss f_ge / (N_g G'), q = w / scale and g the
// weights' gradient:
//
//   balance        dz_e   += s_e h_e (a_e - sum s a)
//   renormalised   dz_i_j += scale q_j h (g_j - sum q g)
//   softmax        dz_e   += scale s_e ([e = i_j] g_j - sum_j q_j g_j)
//   sigmoid        dz_i_j += scale q_j (1 - q_j) g_j
//
// Sums over rows are joined in a fixed order: a block writes one record per
// segment that it meets, and the finishing kernel adds the records in block
// order, so a result does not depend on which block ran first.
#include <math_constants.h>

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
    int64_t per_block;       // rows of one block
};

__device__ __forceinline__ float logistic(float z) { return 1.f / (1.f + expf(-z)); }

// u(z) / u(c): see the head of the file.
__device__ __forceinline__ float ratio(float z, float c, int sigmoid) {
    if (!sigmoid) return expf(z - c);
    return z >= 0.f ? 1.f / (1.f + expf(-z)) : expf(z - c) / (1.f + expf(z));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Order-preserving key of a logit: NaN above all numbers, -0 equal to +0,
// -inf (no expert) and places past E are 0, below every number's key.
__device__ __forceinline__ uint32_t key_of(float z) {
    if (z != z) return 0xffffffffu;
    if (z == -CUDART_INF_F) return 0u;
    const uint32_t b = __float_as_uint(z + 0.f);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    if (key == 0xffffffffu) return CUDART_NAN_F;
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

// Lane l's experts l + 32 i of one row; places past E read -inf.
template <typename T, int V>
__device__ __forceinline__ void load_row(const RouteArgs &a, int64_t t, int lane, float (&z)[V]) {
    const T *row = static_cast<const T *>(a.logits) + t * a.stride;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        z[i] = e < a.experts ? to_float<T>(row[e]) : -CUDART_INF_F;
    }
}

template <int V> __device__ __forceinline__ uint32_t row_peak(const float (&z)[V]) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) best = max(best, key_of(z[i]));
    return __reduce_max_sync(kFull, best);
}

// The top_k largest of the row: lane j gets choice j (index -1 past the last).
template <int V>
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
        if (top == 0) break;
        int first = kMaxExperts;
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
            if (key[i] == top) first = lane + 32 * i;
        first = __reduce_min_sync(kFull, first);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (first == lane + 32 * i) key[i] = 0;
        if (lane == j) {
            index = first;
            value = value_of(top);
        }
    }
}

template <typename T, int V, bool CHOOSE, bool BALANCE>
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
    load_row<T, V>(a, t, lane, z);
    const uint32_t peak = row_peak<V>(z);
    const float top = value_of(peak);
    const float c = a.sigmoid ? fminf(top, 0.f) : top;
    float total = 1.f;
    if (BALANCE || (CHOOSE && !a.renormalize && !a.sigmoid)) {
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            score[i] = ratio(z[i], c, a.sigmoid);
            part += score[i];
        }
        total = warp_sum(part);
    }
    if (CHOOSE) {
        float value, w;
        choose<V>(a, z, lane, index, value);
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
    return peak != 0;
}

// A warp a row.
template <typename T, int V> __global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.tokens;
         t += step) {
        float score[V];
        int index;
        route_row<T, V, true, false>(a, t, lane, score, index);
    }
}

// A block takes per_block rows in a run; its warps share the rows of each
// segment part, and the part's sums become one record.
template <typename T, int V, bool CHOOSE>
__global__ void __launch_bounds__(256) balance_kernel(RouteArgs a) {
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
            if (!route_row<T, V, CHOOSE, true>(a, t, lane, score, index)) continue;
            ++mine;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += score[i];
            if (lane < a.top_k && index >= 0 && index < a.experts) atomicAdd(&counts[index], 1);
        }
        if (lane == 0) atomicAdd(&rows, mine);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane + 32 * i < a.experts) sums[warp * a.experts + lane + 32 * i] = acc[i];
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

// The rows [first, last] of blocks that hold a part of segment g.
__device__ __forceinline__ bool blocks_of(const RouteArgs &a, int g, int64_t &first,
                                          int64_t &last) {
    const int64_t lo = a.offsets ? max(a.offsets[g], 0) : 0;
    const int64_t hi = a.offsets ? min((int64_t)a.offsets[g + 1], a.tokens) : a.tokens;
    if (lo >= hi) return false;
    first = lo / a.per_block;
    last = (hi - 1) / a.per_block;
    return true;
}

// One block: counts, mean scores, the loss, and slope_ge = f_ge / (N_g G').
__global__ void __launch_bounds__(1024)
balance_finish_kernel(RouteArgs a, float *loss, int32_t *counts, float *slope) {
    __shared__ float red[32];
    __shared__ int filled;
    const int tid = threadIdx.x, nt = blockDim.x;
    if (tid == 0) filled = 0;
    __syncthreads();
    int mine = 0;
    for (int g = tid; g < a.segments; g += nt) {
        int64_t b0, b1, n = 0;
        if (!blocks_of(a, g, b0, b1)) continue;
        for (int64_t b = b0; b <= b1; ++b) n += a.rec_rows[b + g];
        mine += n > 0;
    }
    if (mine) atomicAdd(&filled, mine);
    __syncthreads();
    const float share = 1.f / (float)max(filled, 1);
    float part = 0.f;
    for (int g = 0; g < a.segments; ++g) {
        int64_t b0 = 0, b1 = -1, n = 0;
        blocks_of(a, g, b0, b1);
        for (int64_t b = b0; b <= b1; ++b) n += a.rec_rows[b + g];
        const float inv = n > 0 ? 1.f / (float)n : 0.f;
        for (int e = tid; e < a.experts; e += nt) {
            float s = 0.f;
            int64_t c = 0;
            for (int64_t b = b0; b <= b1; ++b) {
                s += a.rec_score[(b + g) * a.experts + e];
                c += a.rec_count[(b + g) * a.experts + e];
            }
            const float f = (float)c * (float)a.experts * inv / (float)a.top_k;
            part += f * s * inv;
            counts[(int64_t)g * a.experts + e] = (int32_t)c;
            slope[(int64_t)g * a.experts + e] = f * inv * share;
        }
    }
    part = warp_sum(part);
    if ((tid & 31) == 0) red[tid >> 5] = part;
    __syncthreads();
    if (tid < 32) {
        part = warp_sum(tid < (nt >> 5) ? red[tid] : 0.f);
        if (tid == 0) *loss = part * share;
    }
}

struct RouteGrad {
    const float *weights;  // gradient of the weights, or null
    const float *slope;    // [segments, experts], or null
    const float *loss;     // the loss's gradient, one value
    void *logits;          // out, [tokens, experts]
};

template <typename T, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteArgs a, RouteGrad d) {
    extern __shared__ float rows[];  // [warps, experts]
    const int lane = threadIdx.x & 31, k = a.top_k;
    float *row = rows + (threadIdx.x >> 5) * a.experts;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    const float up = d.slope ? *d.loss : 0.f;
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.tokens;
         t += step) {
        T *out = static_cast<T *>(d.logits) + t * a.experts;
        uint32_t peak = 0;
        float z[V], dz[V];
        if (!a.mask || a.mask[t]) {
            load_row<T, V>(a, t, lane, z);
            peak = row_peak<V>(z);
        }
        if (peak == 0) {  // no expert: nothing depends on this row
            for (int e = lane; e < a.experts; e += 32) out[e] = from_float<T>(0.f);
            continue;
        }
        const float top = value_of(peak);
        const float c = a.sigmoid ? fminf(top, 0.f) : top;
        const bool dense = d.slope || (d.weights && !a.renormalize && !a.sigmoid);
        float total = 1.f;
        if (dense) {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dz[i] = ratio(z[i], c, a.sigmoid);
                part += dz[i];
            }
            total = warp_sum(part);
        }
        const float inv = 1.f / total;
        // the choice's part: lane j adds `own` at its index, and every expert
        // takes -s_e * shared (softmax that is not renormalised)
        float own = 0.f, shared = 0.f;
        int index = -1;
        if (d.weights) {
            index = lane < k ? a.indices[t * k + lane] : -1;
            if (index >= a.experts) index = -1;
            const float g = index >= 0 ? d.weights[t * k + lane] * a.scale : 0.f;
            const float zi = index >= 0
                ? to_float<T>(static_cast<const T *>(a.logits)[t * a.stride + index])
                : -CUDART_INF_F;
            const float r = index >= 0 ? ratio(zi, c, a.sigmoid) : 0.f;
            const float h = a.sigmoid ? logistic(-zi) : 1.f;
            if (a.renormalize) {
                const float q = r / warp_sum(r);
                const float dot = warp_sum(q * g);
                own = index >= 0 ? q * h * (g - dot) : 0.f;
            } else if (a.sigmoid) {
                own = index >= 0 ? logistic(zi) * h * g : 0.f;
            } else {
                own = r * inv * g;
                shared = warp_sum(own);
            }
        }
        float dot = 0.f;
        const float *slope = nullptr;
        if (d.slope) {
            int64_t end = a.tokens;
            const int g = segment_of(a.offsets, a.segments, t, end);
            if (g >= 0 && g < a.segments) slope = d.slope + (int64_t)g * a.experts;
        }
        if (slope) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = lane + 32 * i;
                if (e < a.experts) dot += dz[i] * inv * slope[e];
            }
            dot = warp_sum(dot);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = lane + 32 * i;
            if (e >= a.experts) continue;
            float v = 0.f;
            if (slope) {
                const float h = a.sigmoid ? logistic(-z[i]) : 1.f;
                v = dz[i] * inv * h * up * (slope[e] - dot);
            }
            if (shared != 0.f) v -= dz[i] * inv * shared;
            row[e] = v;
        }
        __syncwarp();
        if (index >= 0) row[index] += own;
        __syncwarp();
        for (int e = lane; e < a.experts; e += 32) out[e] = from_float<T>(row[e]);
        __syncwarp();
    }
}

struct RouteLayout {
    size_t score, count, rows, total;
    int64_t blocks, per_block;
};

// Blocks of the balance kernel: one per SM, eight rows or more each.
RouteLayout route_layout(int64_t tokens, int64_t experts, int64_t segments) {
    RouteLayout L{};
    L.per_block = (tokens + 147) / 148;
    if (L.per_block < 8) L.per_block = 8;
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

template <typename T, int V>
cudaError_t launch_choice(const RouteArgs &a, int sms, cudaStream_t s) {
    const int64_t want = (a.tokens + 7) / 8;
    const int64_t most = (int64_t)sms * 8;
    route_kernel<T, V><<<(unsigned)(want < most ? want : most), 256, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t launch_balance(const RouteArgs &a, bool choose, int64_t blocks, cudaStream_t s) {
    const size_t smem = (size_t)(8 + 1) * a.experts * 4;
    if (choose) balance_kernel<T, V, true><<<(unsigned)blocks, 256, smem, s>>>(a);
    else balance_kernel<T, V, false><<<(unsigned)blocks, 256, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int V>
cudaError_t launch_backward(const RouteArgs &a, const RouteGrad &d, int sms, cudaStream_t s) {
    const int64_t want = (a.tokens + 7) / 8;
    const int64_t most = (int64_t)sms * 6;
    route_backward_kernel<T, V>
        <<<(unsigned)(want < most ? want : most), 256, (size_t)8 * a.experts * 4, s>>>(a, d);
    return cudaGetLastError();
}

// F(T, V): V values a lane cover E experts.
#define IQK_ROUTE_V(T, F)                      \
    (a.experts <= 64    ? F(T, 2)              \
     : a.experts <= 128 ? F(T, 4)              \
     : a.experts <= 256 ? F(T, 8)              \
     : a.experts <= 512 ? F(T, 16)             \
                        : F(T, 32))
#define IQK_ROUTE_TV(dtype, F)                       \
    ((dtype) == IQK_F32   ? IQK_ROUTE_V(float, F)    \
     : (dtype) == IQK_F16 ? IQK_ROUTE_V(__half, F)   \
                          : IQK_ROUTE_V(__nv_bfloat16, F))

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
#define IQK_F(T, V) launch_choice<T, V>(a, sms, s)
    return cuda_status(IQK_ROUTE_TV(dtype, IQK_F));
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
#define IQK_F(T, V) launch_balance<T, V>(a, weights != nullptr, L.blocks, s)
    if (tokens) err = IQK_ROUTE_TV(dtype, IQK_F);
#undef IQK_F
    if (err != cudaSuccess) return cuda_status(err);
    balance_finish_kernel<<<1, 1024, 0, s>>>(a, loss, counts, slope);
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
#define IQK_F(T, V) launch_backward<T, V>(a, d, sms, s)
    return cuda_status(IQK_ROUTE_TV(dtype, IQK_F));
#undef IQK_F
}

}  // extern "C"
