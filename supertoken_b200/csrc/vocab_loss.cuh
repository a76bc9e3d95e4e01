// What the kernels of the losses over a large vocabulary share (vocab_loss.cu).
#pragma once
#include <limits.h>
#include <stdint.h>

namespace vloss {

typedef unsigned long long u64;
typedef long long i64;

constexpr int PIECE = 256;      // columns per step of the table that finds a row's entries
constexpr int TILE_ROWS = 256;  // the packed rows end on this boundary

// the running maximum starts at a finite value: a logit of -inf then adds 0 to the sum, and one of NaN or +inf makes it NaN
#define LOWEST (-3.0e38f)

struct Meta {
    int counted;          // rows that count
    unsigned int error;   // a wait inside a product ran out
    float out_scale;      // what both gradients are multiplied by in the end
};

struct Plan {
    i64 rows, inner;  // row = outer * inner + inner index
    i64 vocab, dim, dim_padded, rows_padded;
    int k, k_sorted, pieces, parts, reduction, splits;
    bool want_loss, want_grads, hidden_aligned, grad_weight_aligned;
    float temperature, inv_temperature;
    const void *hidden, *weight, *ids, *logits;
    const unsigned char *valid;
    const float *grad_loss;
    i64 hidden_outer, hidden_inner, weight_stride, ids_outer, ids_inner, logits_outer, logits_inner, valid_outer, valid_inner,
        grad_outer, grad_inner;
    int ids_bytes, logits_type;
    // outputs
    float *loss, *lse2;
    void *grad_hidden, *grad_weight;
    // workspace
    Meta *meta;
    int *row_of, *slot_of;   // row of a packed row (-1 behind the last one), packed row of a row (-1: does not count)
    float *plogp;            // sum p log p of a row; NaN: an id outside the vocabulary, a NaN among the teacher's logits
    int2 *entries;           // (id, share) of a row in ascending order of the ids, INT_MAX behind the last one
    unsigned short *first;   // first entry of a row at or behind a piece's first column
    unsigned char *has_entries;
    void *packed;            // counted rows of hidden, one behind another
    const void *weight_rows; // weight, or its copy with rows on 16-byte boundaries
    i64 weight_rows_stride;
    float *part_max, *part_sum, *part_pz, *row_loss;  // [part][packed row]; per row
    float *coef;             // what a packed row of G is multiplied by
    void *g;                 // G of one piece of the vocabulary, [packed row][g_stride]
    i64 g_stride;
    float *acc;              // dH of packed rows in 32 bits, [split][packed row][acc_stride]
    i64 acc_stride;
};

}  // namespace vloss
