// What the kernels of the losses over a large vocabulary share (vocab_loss.cu, vocab_products.cuh).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <stdint.h>

#include "../../include/stbpe.h"

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
    unsigned int tickets; // blocks of the join that are through with their rows
    float in_scale;       // what coef is multiplied by in the end
    float out_scale;      // what both gradients are multiplied by in the end
    int again;            // fixed: a reference was too far from its row's maximum
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
    int2 *refined;           // anew: of a packed row, the entry whose logit is summed once more (-1: none), and its share of the row
    void *packed;            // counted rows of hidden, one behind another
    const void *weight_rows; // weight, or its copy with rows on 16-byte boundaries
    i64 weight_rows_stride;
    float *part_max, *part_sum, *row_loss;  // [part][packed row of the chunk]; per row
    i64 part_stride;
    float *coef;             // what a packed row of dlogits is multiplied by, and in_scale
    // G (16 bits) of one piece of the vocabulary and all packed rows; or (keep) E = exp2(logits - reference) of the whole
    // vocabulary and a chunk of the packed rows, the reference known before (fixed), or each part's own and E to become G
    bool keep, fixed;
    void *g;
    i64 g_stride, chunk_rows;
    float *reference;        // fixed: per packed row
    int *again;              // fixed: [packed row / TILE_ROWS] a reference was too far from the row's maximum; then, per TILE_ROWS rows,
                             // parts that are made again
    float *out_row;          // fixed: what a packed row of dH is multiplied by
    void *scaled;            // fixed: packed rows of the chunk, times coef exp2(reference - lse2)
    float *acc;              // several pieces: dH of packed rows in 32 bits, [packed row][acc_stride]
    float *weight_acc;       // several chunks: dW in 32 bits, [vocab][acc_stride]
    i64 acc_stride;
    int row_blocks;          // blocks that number and pack the rows; those behind them align the weight
    float *split_sums;       // sums of tiles whose depth is split
    unsigned int *split_done;
};

// ---------------------------------------------------------------------------------------------- one row, by one warp
// The tensor cores cut their sums off at each step of 16 terms, always towards 0, so a sum that grows all along, as the logit of a token
// that the row points to does, comes out short by 1e-8 to 1e-7 of itself a step (measured; 5e-6 in bf16 and 1e-5 in fp16 at
// a width of 4 096).  Against that the target's logit, or that of an entry with more than half of the row's share, is summed once
// more in rounded 32 bits, in the loss, in lse and in dlogits, which are small differences of two shares where the model is sure of its
// token (a share about e^-7 below 1 at a width of 4 096 in fp16: dH and dW would be off by 28 % in the 2-norm, and are by 0.1 %).
// The other logits are as short as they are large, and where they are as large as the target's, as logits with an offset in common are, or
// those of several likely tokens, the loss would be off by what the target alone was corrected by.  So lse gets for them what the target
// was short by, of itself, times their mean by shares.  Width 4 096, all logits about 20: the mean loss was 1.8e-4 too small without that and is 1.2e-5 too
// large; losses of 0.04 between likely tokens in fp16: 2.5e-4 too small, 2.2e-5; a target that the row points to, others about 0: 5e-6 too small, 1e-6 too large.
constexpr int REFINED_DIM = 512;
__host__ __device__ __forceinline__ bool refines(const Plan &p) { return !p.few && p.dim > REFINED_DIM; }

// which entry of the row that is, -1: none
__device__ __forceinline__ int refined_entry(const Plan &p, int row, int lane) {
    if (!refines(p)) return -1;
    if (!p.k) return p.entries[row].x != INT_MAX ? 0 : -1;
    int found = -1;
    for (int k = lane; k < p.k; k += 32) {
        const int2 it = p.entries[(i64)row * p.k + k];
        if (it.x != INT_MAX && __int_as_float(it.y) > 0.5f) found = k;
    }
    return __reduce_max_sync(~0u, found);
}

template <class T>
__device__ __forceinline__ float entry_logit(const Plan &p, i64 slot, int row, int k, int lane) {
    const T *w = (const T *)p.weight_rows + p.entries[(i64)row * (p.k ? p.k : 1) + k].x * p.weight_rows_stride, *h = (const T *)p.packed + slot * p.dim_padded;
    float z = 0.f;
#pragma unroll 4
    for (int d = lane * 8; d < p.dim_padded; d += 256) {
        const uint4 x = *(const uint4 *)(h + d), y = *(const uint4 *)(w + d);
        const T *u = (const T *)&x, *v = (const T *)&y;
#pragma unroll
        for (int i = 0; i < 8; ++i) z = fmaf((float)u[i], (float)v[i], z);
    }
    for (int d = 16; d; d >>= 1) z += __shfl_xor_sync(~0u, z, d);
    return z;
}

// The mean of a part's logits by their shares, about: its largest less what shares of 2^side normally distributed logits lie below it on average.  size is
// the logarithm of the part's sum of exponentials about the largest: 0 where that is alone and side where all are as large, when the mean is the
// largest, and a parabola between, less than half a power of e off for any deviation where the largest is up to 1.8 off.  All in powers of 2.
__device__ __forceinline__ float mean_of_part(float top, float size, float side) {
    const float l = fminf(fmaxf(size, 0.f), side);
    return top - 0.18f * l * (side - l);
}

// What follows from a row's lse2 (mean: of its logits, in powers of 2): its loss.  Where E has a fixed reference, the entries in E (from their logits in 32 bits, once
// rounded), the factor of the row's dH and the packed row times it for dW; where each part has its own, G in the place of E.
// m: the row's place in the chunk; slice: which of the row's slices of columns this warp turns into G.
template <class T>
__device__ __forceinline__ void finish_row(const Plan &p, i64 m, i64 slot, int row, float lse2, float mean, float ref, int refined, float target,
                                           int lane, int slice = 0, int slices = 1) {
    const int entries_of_row = p.k ? p.k : 1;
    const float scale = p.inv_temperature * 1.4426950408889634f;
    const int2 *e = p.entries + (i64)row * entries_of_row;
    const float *z = p.entry_z + slot * entries_of_row;
    float longer = 1.f;  // what a teacher's other entries are set right by
    if (refined >= 0) {
        const float before = z[refined], share = exp2f(fmaf(before, scale, -lse2));
        // (a logit of -inf has no share, and no difference to itself)
        if (share > 0.f) lse2 += log1pf(share * expm1f((target - before) * p.inv_temperature)) * 1.4426950408889634f;
        // no more than half a step of 32 bits for each of the sum's (a target near 0 does not tell)
        const float cut = fminf(fmaxf((target - before) / before, 0.f), p.dim * (1.f / 16 / 16777216));
        if (cut > 0.f) lse2 += cut * (mean - share * before * scale), longer += cut;
    }
    const int refined_id = refined >= 0 ? e[refined].x : -1;  // (in more than one entry, if a teacher gives it twice)
    float unit = exp2f(lse2 - ref), minus = ref, times = 1.f;  // a share, the logits and a factor in the units of E
    const i64 from_j = slice == 0 ? 0 : p.vocab * slice / slices / 8 * 8, to_j = slice + 1 == slices ? p.vocab : p.vocab * (slice + 1) / slices / 8 * 8;
    if (p.keep && !p.fixed) {
        unit = 1.f, minus = lse2, times = p.coef[slot] * p.meta->in_scale;
        T *g = (T *)p.g + m * p.g_stride;
        const int shift = 5 + p.group;  // 64 columns to a part, or 128
        constexpr int MANY = 4;  // loads of a lane on their way at a time
        for (i64 j0 = from_j + lane * 8; j0 < to_j; j0 += MANY * 256) {
            uint4 x[MANY];
            float f[MANY];
#pragma unroll
            for (int y = 0; y < MANY; ++y) {
                const i64 j = j0 + y * 256 < to_j ? j0 + y * 256 : j0;
                x[y] = __ldcs((const uint4 *)(g + j)), f[y] = p.part_max[(j >> shift) * p.part_stride + m];
            }
#pragma unroll
            for (int y = 0; y < MANY; ++y) {
                const float by = times * exp2f(f[y] - lse2);
                T *v = (T *)&x[y];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = T((float)v[i] * by);
                if (j0 + y * 256 < to_j) *(uint4 *)(g + j0 + y * 256) = x[y];
            }
        }
        __syncwarp();
    }
    float pz = 0.f, before_rounding = 1.f;
    for (int k = lane; k < entries_of_row; k += 32) {
        const int2 it = e[k];
        if (it.x == INT_MAX) break;
        const float its = it.x == refined_id ? target : z[k] * longer;
        pz += __int_as_float(it.y) * its;
        if (p.keep && it.x >= from_j && it.x < to_j && (k == 0 || e[k - 1].x != it.x)) {  // (the same id again: its first entry takes them all)
            float share = __int_as_float(it.y);
            for (int l = k + 1; l < entries_of_row && e[l].x == it.x; ++l) share += __int_as_float(e[l].y);
            const float value = times * (exp2f(fmaf(its, scale, -minus)) - share * unit);
            const T rounded = T(value);
            ((T *)p.g)[m * p.g_stride + it.x] = rounded;
            if (!p.k && (float)rounded != 0.f) before_rounding = value / (float)rounded;
        }
    }
    for (int d = 16; d; d >>= 1) pz += __shfl_xor_sync(~0u, pz, d);
    if (lane == 0 && slice == 0) {
        const float tau = p.temperature;
        p.lse2[row] = lse2;
        p.row_loss[row] = tau * tau * (lse2 * 0.69314718055994531f + p.plogp[row] - pz * p.inv_temperature);
    }
    if (p.fixed) {
        // The factor of a cross entropy row takes back what its target lost in 16 bits: that is where most of the gradients come from, and the other ids' shares
        // are rounded by as much each (dH 0.0022 to 0.0026 off without it, 0.0017 with it, the result's own rounding; dW 0.0024 to 0.0028 and 0.0021 to
        // 0.0023).  A teacher's entries are rounded each for itself, and an id that one row gives alone would be off by one rounding more.
        const float a = p.coef[slot] * p.meta->in_scale * exp2f(ref - lse2) * __shfl_sync(~0u, before_rounding, 0);
        if (lane == 0) p.out_row[slot] = a * p.meta->out_scale;
        const T *from = (const T *)p.packed + slot * p.dim_padded;
        T *scaled = (T *)p.scaled + m * p.dim_padded;
#pragma unroll 4
        for (int d = lane * 8; d < p.dim_padded; d += 256) {
            uint4 x = *(const uint4 *)(from + d);
            T *v = (T *)&x;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = T((float)v[i] * a);
            *(uint4 *)(scaled + d) = x;
        }
    }
}

// Joins the rows of TILE_ROWS that were made again, one after another.
template <class T>
__device__ __noinline__ void join_again(const Plan &p, i64 r0, i64 m0, i64 n, int lane) {
    for (i64 m = m0; m < m0 + TILE_ROWS && m < n; ++m) {
        const i64 slot = r0 + m;
        const int row = p.row_of[slot];
        const float ref = p.reference[slot];
        float sum = 0.f, logits = 0.f;
        for (int t = lane; t < p.parts; t += 32) {
            const float x = __ldcg(p.part_sum + t * p.part_stride + m);
            const float y = __ldcg(p.part_max + t * p.part_stride + m);
            sum += x, logits += x * mean_of_part(y, log2f(x) + ref - y, 5 + p.group);
        }
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d), logits += __shfl_xor_sync(~0u, logits, d);
        if (sum == INFINITY) sum = NAN;  // a logit of +inf: no other is that far from its reference by now
        const int refined = refined_entry(p, row, lane);
        finish_row<T>(p, m, slot, row, ref + log2f(sum), logits / sum, ref, refined, refined >= 0 ? entry_logit<T>(p, slot, row, refined, lane) : 0.f, lane);
    }
}

// The losses of all rows, in their order, by one warp.  In 64 bits: a lane of 2^20 rows of the same loss rounds 32 768 times the same way in 32,
// 2e-4 of the mean.
__device__ __forceinline__ void add_up(const Plan &p, int lane) {
    double sum = 0.0;
#pragma unroll 16
    for (i64 r = lane; r < p.rows; r += 32) sum += p.row_loss[r];
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    const int n = p.meta->counted;
    if (lane == 0) p.loss[0] = (float)(p.reduction == STBPE_REDUCE_MEAN ? sum / (n > 0 ? n : 1) : sum);
}

}  // namespace vloss
