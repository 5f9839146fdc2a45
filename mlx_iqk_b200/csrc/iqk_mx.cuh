// MXFP4 operators: host-side layout and launchers.
#pragma once

#include "iqk_common.cuh"

namespace iqk {

constexpr int kMxBlock = 32;  // values under one scale

// Workspace of one product, written by its preparation:
//   hdr    [16] int32: [0] routing error bits, [1] work tiles, [2] routable
//          pairs, [3] error bits of the product
//   tickets  int32: parts that are done of each item that CTAs share,
//          per 32 outputs
//   order  [pairs] int32: sorted position -> pair (the others at the tail)
//   place  [pairs, in whole quads] int32: pair -> sorted position, or -1
//   tiles  [max_tiles] int4: {expert, first position, rows (<= cap), 0}
//   codes  [pairs, width / 2], scales [pairs, pitch]: the activations in
//          sorted order
//   slots  f32: shared items' parts (wide rows only)
struct MxLayout {
    size_t hdr, tickets, order, place, tiles, codes, scales, slots, total;
    int64_t max_tiles, pitch;
    int cap, outs;  // rows of a tile, outputs of an item
    __host__ __device__ int zeroed() const { return (int)((order - hdr) / 4); }  // words that start at 0
};

// Rows of this width are wide enough that CTAs may share an item and join its parts.
bool mx_may_join(int64_t width);

MxLayout mx_layout(int64_t pairs, int64_t num_experts, int64_t width, int64_t out_features);

// One call of the product: pairs sorted by expert (order and tiles), or, for a
// single matrix, every row in its own place (order null).
struct MxProduct {
    const uint8_t *codes, *scales;  // the matrices, [experts * out_features] rows
    int64_t scale_stride, out_features, width, pairs, num_experts;
    char *ws;
    MxLayout L;
    bool routed;
    void *y;
    int y_dtype;
};

// The product of few rows in one launch; `state` keeps the counters of shared
// items (0 between calls) and their parts.
struct MxFew {
    const void *x;
    int x_dtype;
    int64_t x_rows, x_stride;
    const int32_t *sel;  // null: one matrix
    int64_t pairs;
    const uint8_t *codes, *scales;
    int64_t scale_stride, num_experts, out_features, width;
    void *y;
    int y_dtype;
    char *state;
};

cudaError_t mx_error_word(int32_t **word);  // on the current device
size_t mx_few_state_bytes(int64_t width);
bool mx_few_fits(int64_t pairs, int64_t num_experts, int64_t out_features, int64_t width,
                 bool routed);
cudaError_t launch_mx_few(const MxFew &p, cudaStream_t stream, int sms);

cudaError_t launch_mx_quantize(const void *x, int dtype, int64_t rows, int64_t width,
                               int64_t row_stride, uint8_t *codes, uint8_t *scales,
                               int64_t scale_stride, const int32_t *place, int copies,
                               int32_t *zero, int zero_words,
                               cudaStream_t stream, int sms);
cudaError_t launch_mx_product(const MxProduct &p, cudaStream_t stream, int sms);

}  // namespace iqk
