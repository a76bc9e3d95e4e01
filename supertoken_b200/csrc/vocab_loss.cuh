// What the kernels of the losses over a large vocabulary share (vocab_loss.cu, vocab_products.cuh).
#pragma once
#include <limits.h>
#include <stdint.h>

namespace vloss {

typedef unsigned long long u64;
typedef long long i64;

constexpr int SMS = 148;
constexpr int PIECE = 256;      // columns per step of the table that finds a row's entries
constexpr int TILE_ROWS = 256;  // packed rows are filled up with zeros to this boundary

// the running maximum starts at a finite value: a logit of -inf then adds 0 to the sum, and one of NaN or +inf makes it NaN
#define LOWEST (-3.0e38f)

// Every kernel is launched while the one before it still runs, and begins by letting the next one come; what it reads and
// writes in memory comes behind before_is_done().
__device__ __forceinline__ void next_may_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void before_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Meta {
    int counted;          // rows that count
    unsigned int tickets; // blocks that are through with their rows' losses
    float in_scale;       // what coef is multiplied by in the end
    float out_scale;      // what both gradients are multiplied by in the end
    int again;            // keep: a reference was too far from its row's maximum
};

struct Plan {
    i64 rows, inner;  // row = outer * inner + inner index
    i64 vocab, dim, dim_padded, rows_padded;
    int k, pieces, parts, reduction, group;
    bool want_loss, want_grads, few;
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
    float *entry_z;          // logits at the entries of a packed row
    void *packed;            // counted rows of hidden, one behind another
    const void *weight_rows; // weight, or its copy with rows on 16-byte boundaries
    i64 weight_rows_stride;
    float *part_max, *part_sum, *row_loss;  // [part][packed row of the chunk]; per row
    i64 part_stride;
    float *coef;             // what a packed row of dlogits is multiplied by, and in_scale
    // G (16 bits) of one piece of the vocabulary and all packed rows; or E = exp2(logits - reference) of the whole
    // vocabulary and a chunk of the packed rows (keep)
    bool keep;
    void *g;
    i64 g_stride, chunk_rows;
    float *reference;        // keep: per packed row
    int *again;              // keep: [packed row / TILE_ROWS] a reference was too far from the row's maximum
    float *out_row;          // keep: what a packed row of dH is multiplied by
    void *scaled;            // keep: packed rows of the chunk, times coef exp2(reference - lse2)
    float *acc;              // several pieces: dH of packed rows in 32 bits, [packed row][acc_stride]
    float *weight_acc;       // several chunks: dW in 32 bits, [vocab][acc_stride]
    i64 acc_stride;
    int row_blocks;          // blocks that number and pack the rows; those behind them align the weight
    float *split_sums;       // sums of tiles whose depth is split
    unsigned int *split_done;
};

}  // namespace vloss
