// Losses over a large vocabulary, straight from the output layer's input: cross entropy, and distillation from a
// teacher's top logits.  With h_i a row of `hidden`, w_j a row of `weight`, s = 1 / temperature and entries
// (t_ik, p_ik) of row i (cross entropy: one, p = 1; s = 1):
//   z_ij = h_i . w_j              lse_i = log sum_j exp(s z_ij)
//   loss_i = T^2 (lse_i + sum_k p_ik (log p_ik - s z_i,t_ik))
//   G_ij = g_i T (exp(s z_ij - lse_i) - sum_k p_ik [j = t_ik])       dH = G W        dW = G^T H
// The N x V logits are never stored.  Two ways to the gradients:
//   keep    (loss and gradients at once): E_ij = exp2(z_ij s log2 e - c_i) goes to memory in 16 bits, for at most 1 GiB of rows (or 2 048
//           of them) at a time, and the sums that make lse_i (lse2_i in powers of 2) beside it.  Three products.
//           With each part's own maximum (of 64 or 128 columns, less 14) as c, E has the range that fp16 needs, and becomes G
//           where it lies once lse_i is known, the entries from z in 32 bits: E is read and written once more (0.2 ms for 4 336 rows of
//           50 257), and G is rounded twice but for the entries, from which most of the gradients come.
//           With c_i = 0 for a row (bf16, where E is above 48 MB and that pass would cost 3 to 6 % of a step) E stays, but for the entries,
//           and a_i = g_i T exp2(c_i - lse2_i) goes to the other factors: dH = a (E W), dW = E^T (a H).  One rounding more
//           reaches dW, 0.0028 off in the 2-norm against 0.0022 with a teacher, where the result's own rounding is 0.0017 (0.0023 where a_i makes up
//           for the target's rounding).  A row whose
//           largest logit lies more than a factor of 2^96 above c_i or 2^80 below gets it as its reference and its tile is made again, which
//           a largest logit between -55 and 66 never needs.
//   anew    (gradients after the loss, as fp16 and losses per row need them through autograd): z is made a second time,
//           and G from it for up to 1 GiB of the vocabulary (or 2 048 ids) at a time, the target's
//           from the logit that the loss had.  Three products behind the loss's one: 3.2 ms for 8 188 x 32 256 x 2 048 in fp16, 2.9 at once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "../../include/stbpe.h"
#include "vocab_products.cuh"

#define STBPE_VISIBLE __attribute__((visibility("default")))

namespace {
using namespace vloss;

// ---------------------------------------------------------------------------------------------- rows and entries
__device__ __forceinline__ i64 load_id(const void *p, int bytes, i64 at) {
    return bytes == 8 ? ((const i64 *)p)[at] : (i64)((const int32_t *)p)[at];
}

__device__ __forceinline__ float load_real(const void *p, int type, i64 at) {
    if (type == STBPE_REAL_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[at]);
    if (type == STBPE_REAL_FP16) return __half2float(((const __half *)p)[at]);
    return ((const float *)p)[at];
}

// One warp per row: softmax of the teacher's entries in 32 bits, entries in ascending order of their ids (the order in
// which the products meet them), and for each piece of columns the first entry that lies in it or behind.  The ids
// come in the order of the logits; 64-bit words (id, share), ITEMS to a lane, are ordered by a bitonic network of shuffles.
// Floor: 8 to 12 bytes per entry.
template <int ITEMS>
__global__ void __launch_bounds__(128) teacher_kernel(Plan p) {
    next_may_come();
    before_is_done();
    __shared__ u64 sorted[4][ITEMS * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 *e = sorted[warp];
    for (i64 row = (i64)blockIdx.x * 4 + warp; row < p.rows; row += (i64)gridDim.x * 4) {
        const i64 o = (unsigned)row / (unsigned)p.inner, i = row - o * p.inner;
        const i64 id_at = o * p.ids_outer + i * p.ids_inner, real_at = o * p.logits_outer + i * p.logits_inner;
        i64 id[ITEMS];
        float t[ITEMS];
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            const int k = x * 32 + lane;
            id[x] = k < p.k ? load_id(p.ids, p.ids_bytes, id_at + k) : -1;
            t[x] = k < p.k ? load_real(p.logits, p.logits_type, real_at + k) : 0.f;
        }
        float top = -INFINITY, sum = 0.f, plogp = 0.f;
        bool bad = false;
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            if (id[x] < 0) continue;
            bad |= id[x] >= p.vocab || isnan(t[x]) || t[x] == INFINITY;
            top = fmaxf(top, t[x]);
        }
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        bool nan = false;
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) nan |= id[x] >= 0 && isnan(t[x]);
        bad = __any_sync(~0u, bad), nan = __any_sync(~0u, nan);
        const bool counted = top > -INFINITY || nan;
        // the difference first: a logit times 1 / temperature may leave the range of 32 bits, and the maximum less itself is 0
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            t[x] = (t[x] - top) * p.inv_temperature;
            if (id[x] >= 0 && counted) sum += expf(t[x]);
        }
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        const float inv = 1.f / sum, log_sum = logf(sum);
        u64 word[ITEMS];
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            word[x] = ~0ull;  // no entry: behind all others
            if (id[x] < 0 || !counted || bad) continue;
            const float share = expf(t[x]) * inv;
            if (share > 0.f) {
                plogp += share * (t[x] - log_sum);
                word[x] = ((u64)id[x] << 32) | __float_as_uint(share);
            }
        }
        for (int d = 16; d; d >>= 1) plogp += __shfl_xor_sync(~0u, plogp, d);
#pragma unroll
        for (int size = 2; size <= ITEMS * 32; size <<= 1) {
#pragma unroll
            for (int step = size >> 1; step; step >>= 1) {
                if (step >= 32) {
#pragma unroll
                    for (int x = 0; x < ITEMS; ++x) {
                        const int y = x ^ (step >> 5);
                        if (y < x) continue;
                        const bool up = !((x * 32) & size);
                        if ((word[x] > word[y]) == up) {
                            const u64 w = word[x];
                            word[x] = word[y], word[y] = w;
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < ITEMS; ++x) {
                        const u64 w = __shfl_xor_sync(~0u, word[x], step);
                        const bool up = !((x * 32 + lane) & size), low = !(lane & step);
                        // the lower place of an ascending pair keeps the smaller word
                        if ((w < word[x]) == (up == low)) word[x] = w;
                    }
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            const int k = x * 32 + lane;
            e[k] = word[x];
            if (k < p.k) p.entries[row * p.k + k] = word[x] == ~0ull ? make_int2(INT_MAX, 0) : make_int2((int)(word[x] >> 32), (int)word[x]);
        }
        __syncwarp();
        for (int t = lane; t < p.pieces; t += 32) {  // first entry at or behind the piece's first column
            const u64 from = (u64)t * PIECE << 32;
            int at = 0;
#pragma unroll
            for (int step = ITEMS * 16; step; step >>= 1)
                if (e[at + step - 1] < from) at += step;
            if (at < ITEMS * 32 && e[at] < from) ++at;
            p.first[row * p.pieces + t] = (unsigned short)(at < p.k ? at : p.k);
        }
        if (lane == 0) {
            p.plogp[row] = bad ? NAN : plogp;
            p.has_entries[row] = counted;
        }
    }
}

// 16-bit numbers of one row by one warp: 16, 4 or 2 bytes at a time as both rows allow, zeros from `inside` up to `all`.
template <class T>
__device__ __forceinline__ void copy_row(T *to, const T *from, i64 inside, i64 all, int lane) {
    const uintptr_t at = (uintptr_t)to | (uintptr_t)from;
    if (at % 16 == 0 && inside % 8 == 0 && all == inside) {
#pragma unroll 4
        for (i64 d = lane * 8; d < inside; d += 256) *(uint4 *)(to + d) = *(const uint4 *)(from + d);
    } else if (at % 4 == 0) {
#pragma unroll 16
        for (i64 d = lane * 2; d < all; d += 64) {
            const uint32_t both = d + 1 < inside ? *(const uint32_t *)(from + d) : d < inside ? *(const unsigned short *)(from + d) : 0u;
            if (d + 1 < all) *(uint32_t *)(to + d) = both;
            else *(unsigned short *)(to + d) = (unsigned short)both;
        }
    } else {
#pragma unroll 8
        for (i64 d = lane; d < all; d += 32) to[d] = d < inside ? from[d] : T(0.f);
    }
}

// Which rows count, in their order (row_of, slot_of); the entry of a cross entropy row; what each counted row's dlogits are
// multiplied by.  Every block has a range of the rows and counts by itself those that count before it, and all of them, eight loads
// of a thread on their way at a time, so that no launch lies between the rows' numbers and what follows.
// Then counted rows of `hidden` go one behind another, zeros up to the end of the last tile, a warp to a row: products then do no
// work for padding, never multiply what a masked row holds (it may be NaN), and may read rows of any stride or alignment.  The
// rows of dH that do not count get their zeros here.
// dlogits are held in the inputs' 16-bit type, so they are brought into that type's range: the largest |g_i T| becomes 16376 (in the rows where |g_i| is
// near the largest fp16 keeps shares down to 2^-28 at full precision; a row with 2^-20 of it keeps those down to 2^-8, and 2^-18 coarsely;
// its entries stay below 2^15; just below a power of two, a target's
// dlogit, -g T (1 - q), loses half as much to its rounding as just above one), and both gradients are scaled back in 32 bits.
template <class T>
__global__ void __launch_bounds__(1024) rows_kernel(Plan p) {
    next_may_come();
    before_is_done();
    if (blockIdx.x >= p.row_blocks) {  // a weight whose rows do not start on 16-byte boundaries is copied so that they do
        const i64 blocks = gridDim.x - p.row_blocks;
        for (i64 j = blockIdx.x - p.row_blocks + (threadIdx.x >> 5) * blocks; j < p.vocab; j += blocks * 32)
            copy_row((T *)p.weight_rows + j * p.dim_padded, (const T *)p.weight + j * p.weight_stride, p.dim, p.dim_padded, threadIdx.x & 31);
        return;
    }
    __shared__ int befores[32], alls[32], in_warp[32], slots[1024];
    __shared__ float mosts[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 each_block = (p.rows + p.row_blocks - 1) / p.row_blocks;
    const i64 start = blockIdx.x * each_block, end = start + each_block < p.rows ? start + each_block : p.rows;
    const bool last = blockIdx.x == p.row_blocks - 1;
    const bool each = p.want_grads && p.reduction == STBPE_REDUCE_NONE && p.grad_loss;
    const float one = p.want_grads && p.grad_loss && !each && p.rows > 0 ? p.grad_loss[0] : 1.f;
    auto counts = [&](i64 row, i64 &id) {
        const i64 o = (unsigned)row / (unsigned)p.inner, i = row - o * p.inner;
        const bool there = !p.valid || p.valid[o * p.valid_outer + i * p.valid_inner];
        if (p.k) return there && p.has_entries[row];
        id = load_id(p.ids, p.ids_bytes, o * p.ids_outer + i * p.ids_inner);
        return there && id >= 0;
    };
    auto grad_of = [&](i64 row) {
        const i64 o = (unsigned)row / (unsigned)p.inner, i = row - o * p.inner;
        return p.grad_loss[o * p.grad_outer + i * p.grad_inner];
    };
    int before = 0, all = 0;
    float most = each ? 0.f : fabsf(one);
#pragma unroll 8
    for (i64 row = threadIdx.x; row < p.rows; row += 1024) {
        i64 id;
        const bool counted = counts(row, id);
        all += counted, before += counted && row < start;
        if (each && last && counted) most = fmaxf(most, fabsf(grad_of(row)));
    }
    for (int d = 16; d; d >>= 1) {
        before += __shfl_xor_sync(~0u, before, d), all += __shfl_xor_sync(~0u, all, d);
        most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    }
    if (lane == 0) befores[warp] = before, alls[warp] = all, mosts[warp] = most;
    __syncthreads();
    before = befores[lane], all = alls[lane], most = mosts[lane];
    for (int d = 16; d; d >>= 1) {
        before += __shfl_xor_sync(~0u, before, d), all += __shfl_xor_sync(~0u, all, d);
        most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    }
    const i64 n = all, until = (n + TILE_ROWS - 1) / TILE_ROWS * TILE_ROWS;
    for (i64 r0 = start; r0 < end; r0 += 1024) {
        const i64 row = r0 + threadIdx.x;
        i64 id = -1;
        const bool there = row < end, counted = there && counts(row, id);
        const unsigned votes = __ballot_sync(~0u, counted);
        if (lane == 0) in_warp[warp] = __popc(votes);
        __syncthreads();
        int slot = lane < warp ? in_warp[lane] : 0, whole = in_warp[lane];
        for (int d = 16; d; d >>= 1) slot += __shfl_xor_sync(~0u, slot, d), whole += __shfl_xor_sync(~0u, whole, d);
        slot += before + __popc(votes & ((1u << lane) - 1));
        before += whole;
        slots[threadIdx.x] = counted ? slot : -1;
        if (there) {
            p.slot_of[row] = counted ? slot : -1;
            const bool outside = !p.k && id >= p.vocab;
            float nan = outside ? NAN : 0.f;
            if (p.k) {
                nan = p.plogp[row] * 0.f;
            } else {
                p.entries[row] = make_int2(outside || id < 0 ? INT_MAX : (int)id, __float_as_int(1.f));
                p.plogp[row] = nan;
            }
            if (counted) {
                p.row_of[slot] = (int)row;
                if (p.want_grads) p.coef[slot] = (each ? grad_of(row) : 1.f) + nan;
            } else if (p.want_loss) {
                p.row_loss[row] = p.lse2[row] = 0.f;
            }
        }
        __syncthreads();
        const i64 here = end - r0 < 1024 ? end - r0 : 1024;
        for (i64 y = warp; y < here; y += 32) {
            const i64 its = r0 + y;
            const int to = slots[y];
            if (to >= 0) {
                const i64 o = (unsigned)its / (unsigned)p.inner, i = its - o * p.inner;
                copy_row((T *)p.packed + (i64)to * p.dim_padded, (const T *)p.hidden + o * p.hidden_outer + i * p.hidden_inner, p.dim,
                         p.dim_padded, lane);
            } else if (p.grad_hidden) {
                T *at = (T *)p.grad_hidden + its * p.dim;
                if (p.dim % 8 == 0)
                    for (int d = lane * 8; d < p.dim; d += 256) *(uint4 *)(at + d) = make_uint4(0, 0, 0, 0);
                else
                    for (int d = lane; d < p.dim; d += 32) at[d] = T(0.f);
            }
        }
        __syncthreads();
    }
    for (i64 c = n + blockIdx.x + warp * p.row_blocks; c < until; c += p.row_blocks * 32)
        for (int d = lane * 8; d < p.dim_padded; d += 256) *(uint4 *)((T *)p.packed + c * p.dim_padded + d) = make_uint4(0, 0, 0, 0);
    const i64 step = (i64)p.row_blocks * 1024;
    for (i64 c = n + blockIdx.x * 1024 + threadIdx.x; c < p.rows_padded; c += step) p.row_of[c] = -1;
    if (p.fixed) {
        for (i64 c = blockIdx.x * 1024 + threadIdx.x; c < p.rows_padded; c += step) p.reference[c] = 0.f;
        for (i64 c = blockIdx.x * 1024 + threadIdx.x; c < 2 * p.rows_padded / TILE_ROWS; c += step) p.again[c] = 0;
    }
    if (!last) return;
    if (p.split_done)
        for (int x = threadIdx.x; x < 2 * SMS * 8; x += 1024) p.split_done[x] = 0;
    if (threadIdx.x == 0) {
        const float factor = p.temperature / (p.reduction == STBPE_REDUCE_MEAN ? (float)(n > 0 ? n : 1) : 1.f);
        // (in times factor is finite where all are 0, too)
        const float in = 16376.f / fminf(fmaxf(most * factor, 1e-25f), 1e30f);
        p.meta->counted = (int)n, p.meta->tickets = 0, p.meta->again = 0;
        p.meta->in_scale = (each ? 1.f : one) * factor * in;
        p.meta->out_scale = 1.f / in;
    }
}

// The losses of up to eight rows, as when text is scored as it is generated: bound by the weight, which is read once (V D 2 bytes), and by
// launches, so numbering the rows and the product are one kernel.  A warp takes four of the weight's rows at a time, a lane 16 bytes of each per
// 256 columns, against the rows of `hidden` in shared memory; sums in 32 bits, every block leaves its part as the tiles
// of a product do.  17 MB of weight in 6 us, 12 to 14 us a captured call where the tensor cores' tiles of 128 rows and a launch more take 18.
constexpr int FEW_ROWS = 8, FEW_NUMBERS = 16384;  // rows, and rows (rounded up to a power of two) times width
template <class T, int ROWS>
__global__ void __launch_bounds__(256) few_kernel(Plan p) {
    next_may_come();
    before_is_done();
    __shared__ __align__(16) T h[FEW_NUMBERS];
    __shared__ int ids[FEW_ROWS], slots[FEW_ROWS];
    __shared__ float tops[8][FEW_ROWS], sums[8][FEW_ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool first = blockIdx.x == 0;
    const i64 warps = (i64)gridDim.x * 8;
    // the weight's first rows come while the other inputs are looked at
    for (int x = 0; x < 4; ++x) {
        const i64 j = (i64)blockIdx.x * 8 + warp + x * warps;
        if (j >= p.vocab) break;
        for (int d = lane * 64; d < p.dim; d += 2048)
            asm volatile("prefetch.global.L2 [%0];" ::"l"((const T *)p.weight_rows + j * p.weight_rows_stride + d));
    }
    if (warp == 0) {
        bool counted = false, outside = false;
        i64 id = -1;
        if (lane < p.rows) {
            const i64 o = (unsigned)lane / (unsigned)p.inner, i = lane - o * p.inner;
            id = load_id(p.ids, p.ids_bytes, o * p.ids_outer + i * p.ids_inner);
            counted = id >= 0 && (!p.valid || p.valid[o * p.valid_outer + i * p.valid_inner]);
            outside = id >= p.vocab;
        }
        const unsigned votes = __ballot_sync(~0u, counted);
        const int slot = counted ? __popc(votes & ((1u << lane) - 1)) : -1;
        if (lane < FEW_ROWS) slots[lane] = slot, ids[lane] = outside || !counted ? -1 : (int)id;
        if (first && lane < p.rows) {
            p.slot_of[lane] = slot;
            p.entries[lane] = make_int2(!counted || outside ? INT_MAX : (int)id, __float_as_int(1.f));
            p.plogp[lane] = outside ? NAN : 0.f;
            if (counted) p.row_of[slot] = lane;
            else p.row_loss[lane] = p.lse2[lane] = 0.f;
        }
        if (first && lane == 0) p.meta->counted = __popc(votes), p.meta->tickets = 0, p.meta->again = 0;
    }
    // rows that do not count take part in what nobody reads
    for (int r = warp; r < ROWS; r += 8) {
        const i64 row = r < p.rows ? r : 0, o = (unsigned)row / (unsigned)p.inner, i = row - o * p.inner;
        copy_row(h + r * p.dim, (const T *)p.hidden + o * p.hidden_outer + i * p.hidden_inner, p.dim, p.dim, lane);
    }
    __syncthreads();
    const float scale = 1.4426950408889634f;
    float top[ROWS], sum[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) top[r] = LOWEST, sum[r] = 0.f;
    for (i64 j0 = (i64)blockIdx.x * 8 + warp; j0 < p.vocab; j0 += 4 * warps) {
        float z[4][ROWS];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) z[x][r] = 0.f;
#pragma unroll 2
        for (int d = lane * 8; d < p.dim; d += 256) {
            uint4 w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                w[x] = j0 + x * warps < p.vocab ? __ldcs((const uint4 *)((const T *)p.weight_rows + (j0 + x * warps) * p.weight_rows_stride + d))
                                                : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const uint4 u = *(const uint4 *)(h + r * p.dim + d);
                const T *a = (const T *)&u;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const T *b = (const T *)&w[x];
#pragma unroll
                    for (int i = 0; i < 8; ++i) z[x][r] = fmaf((float)a[i], (float)b[i], z[x][r]);
                }
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const i64 j = j0 + x * warps;
            if (j >= p.vocab) break;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                for (int d = 16; d; d >>= 1) z[x][r] += __shfl_xor_sync(~0u, z[x][r], d);
                if (lane == 0 && ids[r] == j) p.entry_z[slots[r]] = z[x][r];
                const float now = fmaxf(top[r], z[x][r] * scale);
                sum[r] = sum[r] * exp2f(top[r] - now) + exp2f(fmaf(z[x][r], scale, -now));
                top[r] = now;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (lane == 0) tops[warp][r] = top[r], sums[warp][r] = sum[r];
    __syncthreads();
    if (threadIdx.x < ROWS && slots[threadIdx.x] >= 0) {
        float t = tops[0][threadIdx.x], s = sums[0][threadIdx.x];
        for (int w = 1; w < 8; ++w) {
            const float m = tops[w][threadIdx.x], both = fmaxf(t, m);
            s = s * exp2f(t - both) + sums[w][threadIdx.x] * exp2f(m - both);
            t = both;
        }
        const i64 to = blockIdx.x * p.part_stride + slots[threadIdx.x];
        p.part_max[to] = t, p.part_sum[to] = s;
    }
}

// ---------------------------------------------------------------------------------------------- after the products
// Eight rows of a chunk (and a slice of their columns, where few rows are turned into G) to a block: joins what the parts of the columns left, in a fixed order (eight threads read a sector, 32 parts
// at a time), to lse and the loss of a row; then a warp has a row.  Where E is kept, the row's E gets its entries and the packed row its factor.
// all_blocks: of the joins of all chunks, the last of which adds up.
template <class T>
__global__ void __launch_bounds__(256) join_kernel(Plan p, i64 r0, i64 rows, int slices, unsigned all_blocks) {
    next_may_come();
    before_is_done();
    __shared__ float tops[8][8], sums[8][8], logits[8][8], lse2s[8], means[8], refs[8];
    __shared__ double losses[8];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 counted = p.meta->counted;
    const i64 n = counted - r0 < 0 ? 0 : counted - r0 < rows ? counted - r0 : rows;
    const i64 until = p.fixed ? (n + TILE_ROWS - 1) / TILE_ROWS * TILE_ROWS : n;
    const int slice = blockIdx.x % slices;
    for (i64 m0 = (i64)(blockIdx.x / slices) * 8; m0 < until; m0 += (i64)(gridDim.x / slices) * 8) {
        float top = LOWEST, sum = 0.f, logit = 0.f;  // of the row's parts: maximum, sum of exp, that times the mean logit
        auto add = [&](float m, float x, float y) {
            const float both = fmaxf(top, m);
            if (p.fixed) {  // all parts of a row have the same reference
                sum += x, logit += y;
            } else {
                const float f = exp2f(top - both), g = exp2f(m - both);
                sum = sum * f + x * g, logit = logit * f + y * g;
            }
            top = both;
        };
        const float shift = p.keep && !p.fixed ? 14.f : 0.f, side = 5 + p.group;  // (MAKE_R: what the maxima are less by; 2^6 columns to a part, or 2^7)
        // the row of this warp; the sum of its target's logit needs nothing of the parts
        const i64 m = m0 + warp, slot = r0 + m;
        const int row = m < n ? p.row_of[slot] : 0;
        const int refined = m < n ? refined_entry(p, row, lane) : -1;
        float sum_z = 0.f;
        if (m0 + (lane & 7) < n) {
            const float *from_max = p.part_max + m0 + (lane & 7), *from_sum = p.part_sum + m0 + (lane & 7);
#pragma unroll 4
            for (int t = warp * 4 + (lane >> 3); t < p.parts; t += 32) {
                const float m = from_max[t * p.part_stride], x = from_sum[t * p.part_stride];
                add(m, x, refines(p) ? x * mean_of_part(m + shift, log2f(x) - (p.fixed ? m : shift), side) : 0.f);
            }
        }
        for (int d = 8; d < 32; d <<= 1) {
            const float m = __shfl_xor_sync(~0u, top, d), x = __shfl_xor_sync(~0u, sum, d), y = __shfl_xor_sync(~0u, logit, d);
            add(m, x, y);
        }
        if (refined >= 0) sum_z = entry_logit<T>(p, slot, row, refined, lane);
        if (lane < 8) tops[warp][lane] = top, sums[warp][lane] = sum, logits[warp][lane] = logit;
        __syncthreads();
        if (threadIdx.x < 8) {
            top = tops[0][lane], sum = sums[0][lane], logit = logits[0][lane];
            for (int w = 1; w < 8; ++w) add(tops[w][lane], sums[w][lane], logits[w][lane]);
            float ref = top;
            // a logit of +inf makes the sum NaN about a maximum, and has to about a fixed reference
            if (p.fixed && top == INFINITY) sum = NAN;
            if (p.fixed && m0 + lane < n) {
                ref = p.reference[r0 + m0 + lane];
                // above, exp2 must not overflow; below, 2^-126 is the least that is kept, 2^-46 of the maximum then: 2^-25 of it for 2^21 ids
                const float above = top - ref;
                if ((above > 96.f || above < -80.f) && fabsf(top) < INFINITY) {
                    p.reference[r0 + m0 + lane] = top;
                    p.again[(r0 + m0) / TILE_ROWS] = p.meta->again = 1;
                }
            }
            refs[lane] = ref, lse2s[lane] = ref + log2f(sum), means[lane] = logit / sum;
        }
        __syncthreads();
        T *scaled = (T *)p.scaled + m * p.dim_padded;
        if (m < n) {
            finish_row<T>(p, m, slot, row, lse2s[warp], means[warp], refs[warp], refined, sum_z, lane, slice, slices);
        } else if (p.fixed && m < until) {  // zeros behind the last row
            for (int d = lane * 8; d < p.dim_padded; d += 256) *(uint4 *)(scaled + d) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    if (p.reduction == STBPE_REDUCE_NONE || p.keep) return;  // (keep: a row may be made again, the launch for the gradients adds up)
    // the block that is through last adds the losses up, in the order of the rows
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&p.meta->tickets, 1u) == all_blocks - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double sum = 0.0;  // (as in add_up)
#pragma unroll 8
    for (i64 r = threadIdx.x; r < p.rows; r += 256) sum += __ldcg(p.row_loss + r);
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) losses[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < 8; ++w) all += losses[w];
        p.loss[0] = (float)(p.reduction == STBPE_REDUCE_MEAN ? all / (counted > 0 ? counted : 1) : all);
    }
}

// Gradients after the loss: the refined entry of a packed row and its share, a warp to a row.  Among entries of the same id it is the first, where G
// takes the whole share.  Bound by the memory that the rows and their targets' rows of the weight come from.
template <class T>
__global__ void __launch_bounds__(256) refine_kernel(Plan p) {
    next_may_come();
    before_is_done();
    const int lane = threadIdx.x & 31, n = p.meta->counted;
    const float scale = p.inv_temperature * 1.4426950408889634f;
    for (i64 slot = (i64)blockIdx.x * 8 + (threadIdx.x >> 5); slot < n; slot += (i64)gridDim.x * 8) {
        const int row = p.row_of[slot];
        int k = refined_entry(p, row, lane);
        const float z = k >= 0 ? entry_logit<T>(p, slot, row, k, lane) : 0.f;
        const int2 *e = p.entries + (i64)row * (p.k ? p.k : 1);
        while (k > 0 && e[k - 1].x == e[k].x) --k;
        if (lane == 0) p.refined[slot] = make_int2(k, __float_as_int(exp2f(fmaf(z, scale, -p.lse2[row]))));
    }
}

// What comes down to the loss, onto gradients that were made with it.
__global__ void __launch_bounds__(256) scale_kernel(__nv_bfloat16 *a, i64 n_a, __nv_bfloat16 *b, i64 n_b, const float *by) {
    next_may_come();
    before_is_done();
    const float f = *by;
    if (f == 1.f) return;
    for (int which = 0; which < 2; ++which) {
        __nv_bfloat16 *p = which ? b : a;
        const i64 n = which ? n_b : n_a;
        for (i64 x = ((i64)blockIdx.x * 256 + threadIdx.x) * 8; x < n; x += (i64)gridDim.x * 2048) {
            if (x + 8 <= n) {
                uint4 v = *(uint4 *)(p + x);
                __nv_bfloat16 *e = (__nv_bfloat16 *)&v;
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = __float2bfloat16(__bfloat162float(e[i]) * f);
                *(uint4 *)(p + x) = v;
            } else {
                for (i64 i = x; i < n; ++i) p[i] = __float2bfloat16(__bfloat162float(p[i]) * f);
            }
        }
    }
}

// dH of several pieces in the caller's rows and type, zeros where a row does not count.
template <class T>
__global__ void __launch_bounds__(256) scatter_kernel(Plan p) {
    next_may_come();
    before_is_done();
    const float scale = p.meta->out_scale;
    const i64 total = p.rows * p.dim;
    for (i64 x = (i64)blockIdx.x * 256 + threadIdx.x; x < total; x += (i64)gridDim.x * 256) {
        const i64 row = x / p.dim, d = x - row * p.dim;
        const int c = p.slot_of[row];
        ((T *)p.grad_hidden)[x] = T(c < 0 ? 0.f : p.acc[c * p.acc_stride + d] * scale);
    }
}

// ---------------------------------------------------------------------------------------------- host
#define VCK(call)                                                                              \
    do {                                                                                       \
        cudaError_t c_ = (call);                                                               \
        if (c_ != cudaSuccess) return fail(err, err_len, STBPE_E_CUDA, #call, cudaGetErrorString(c_)); \
    } while (0)

#define VTRY(call)                        \
    do {                                  \
        const int st_ = (call);           \
        if (st_ != STBPE_OK) return st_;  \
    } while (0)

int fail(char *err, size_t len, int status, const char *what, const char *why) {
    if (err && len) snprintf(err, len, "%s: %s", what, why);
    if (status == STBPE_E_CUDA) cudaGetLastError();
    return status;
}

i64 up_to(i64 x, i64 unit) { return (x + unit - 1) / unit * unit; }

// CTAs to a tile of a product, by what it takes: steps of 64 terms, 0.36 us for 256 x 256 by a pair and 0.28 for 128 x 128 by a single
// CTA, of which twice as many run at a time: 1.7 against 1.1 PFLOP/s in a launch of few rounds (in long ones 1.5 to 1.6 against 0.93 to 0.98).
int group_of(i64 rows, i64 cols, i64 rows2, i64 cols2, i64 depth, i64 depth2, bool split, bool split2) {
    double cost[3];
    for (int g = 1; g <= 2; ++g) {
        const i64 side = 128 * g;
        const unsigned tiles[2] = {(unsigned)(((rows + side - 1) / side) * ((cols + side - 1) / side)),
                                   (unsigned)(((rows2 + side - 1) / side) * ((cols2 + side - 1) / side))};
        const unsigned steps[2] = {(unsigned)((depth + 63) / 64), (unsigned)((depth2 + 63) / 64)};
        cost[g] = (double)deal(tiles, steps, {split, split2}, SMS / g).steps * (g == 2 ? 0.36 : 0.28);
    }
    return cost[1] < cost[2] ? 1 : 2;
}

// Checks the arguments and lays the workspace out; `bytes` gets its size.
int plan(const stbpe_vocab_loss *a, Plan &p, i64 &bytes, char *err, size_t err_len) {
    auto bad = [&](const char *why) { return fail(err, err_len, STBPE_E_BADARG, "stbpe_vocab_loss", why); };
    if (!a) return bad("no arguments");
    if (a->outer < 0 || a->inner < 0 || a->vocab < 1 || a->dim < 1) return bad("negative or empty size");
    if (a->vocab > INT_MAX - 65536 || a->dim > (1 << 20)) return bad("vocabulary or width too large");
    if (a->inner && a->outer > (INT_MAX - 65536) / a->inner) return bad("too many rows");
    const i64 tall = (a->outer * a->inner + 127) / 128, wide = (a->vocab + 127) / 128, deep = (a->dim + 127) / 128;
    if (tall * wide > INT_MAX / 4 || wide * deep > INT_MAX / 4 || tall * deep > INT_MAX / 4 || wide > INT_MAX / 128)
        return bad("too many rows for this vocabulary and width");
    if (a->type != STBPE_REAL_BF16 && a->type != STBPE_REAL_FP16) return bad("hidden and weight are bf16 or fp16");
    if (a->k < 0 || a->k > STBPE_VOCAB_LOSS_MAX_K) return bad("number of teacher entries out of range");
    if (a->ids_bytes != 4 && a->ids_bytes != 8) return bad("ids have 4 or 8 bytes");
    if (a->k && (a->logits_type < STBPE_REAL_BF16 || a->logits_type > STBPE_REAL_FP32)) return bad("type of the teacher's logits");
    // below, logits over it leave the 24 bits that a difference of theirs is taken in; above, its square and the gradients' scale the exponents of 32
    if (!(a->temperature >= STBPE_MIN_TEMPERATURE && a->temperature <= STBPE_MAX_TEMPERATURE)) return bad("temperature is between 2^-16 and 2^16");
    if (!a->k && a->temperature != 1.f) return bad("cross entropy has no temperature");
    if (a->reduction < STBPE_REDUCE_NONE || a->reduction > STBPE_REDUCE_MEAN) return bad("reduction");
    if (!(a->want & (STBPE_WANT_LOSS | STBPE_WANT_GRADS))) return bad("nothing is wanted");
    p = Plan{};
    p.rows = a->outer * a->inner, p.inner = a->inner > 0 ? a->inner : 1;
    p.vocab = a->vocab, p.dim = a->dim, p.k = a->k;
    p.dim_padded = up_to(a->dim, 8);
    p.rows_padded = up_to(p.rows > 0 ? p.rows : 1, TILE_ROWS);
    p.pieces = (int)((a->vocab + PIECE - 1) / PIECE);
    p.row_blocks = p.rows + TILE_ROWS <= 16 * SMS ? (int)(p.rows + TILE_ROWS) / 16 : SMS;
    p.temperature = a->temperature, p.inv_temperature = 1.f / a->temperature;
    p.reduction = a->reduction;
    p.want_loss = (a->want & STBPE_WANT_LOSS) != 0, p.want_grads = (a->want & STBPE_WANT_GRADS) != 0;
    p.hidden = a->hidden, p.hidden_outer = a->hidden_outer, p.hidden_inner = a->hidden_inner;
    p.weight = a->weight, p.weight_stride = a->weight_stride;
    p.ids = a->ids, p.ids_bytes = a->ids_bytes, p.ids_outer = a->ids_outer, p.ids_inner = a->ids_inner;
    p.logits = a->logits, p.logits_type = a->logits_type, p.logits_outer = a->logits_outer, p.logits_inner = a->logits_inner;
    p.valid = a->valid, p.valid_outer = a->valid_outer, p.valid_inner = a->valid_inner;
    p.grad_loss = a->grad_loss, p.grad_outer = a->grad_outer, p.grad_inner = a->grad_inner;
    p.loss = a->loss, p.lse2 = a->lse2, p.grad_hidden = a->grad_hidden, p.grad_weight = a->grad_weight;
    const bool aligned = (uintptr_t)a->weight % 16 == 0 && a->weight_stride % 8 == 0 && a->weight_stride >= a->dim && a->dim % 8 == 0;
    p.weight_rows_stride = aligned ? a->weight_stride : p.dim_padded;
    if (!aligned && p.row_blocks > SMS / 4) p.row_blocks = SMS / 4;  // (the others align the weight: a block of either kind has an SM)
    // at most KEPT bytes of E, G or parts' sums at a time (for large vocabularies 2048 rows of E or sums, for many rows 2048 columns of G)
    constexpr i64 KEPT = 1ll << 30, FIXED_BYTES = 48ll << 20;
    const i64 all = up_to(a->vocab, PIECE);
    p.keep = p.want_loss && p.want_grads;
    p.chunk_rows = p.rows_padded, p.g_stride = all;
    if (p.keep) {
        const i64 most = KEPT / (2 * all) / TILE_ROWS * TILE_ROWS;
        p.chunk_rows = p.rows_padded <= most ? p.rows_padded : most > 2048 ? most : p.rows_padded < 2048 ? p.rows_padded : 2048;
    } else if (!p.want_grads) {
        const i64 most = KEPT / (8 * ((a->vocab + 63) / 64)) / TILE_ROWS * TILE_ROWS, least = most > 2048 ? most : 2048;
        if (p.chunk_rows > least) p.chunk_rows = least;
    } else {
        const i64 most = KEPT / (2 * p.rows_padded) / PIECE * PIECE;
        p.g_stride = all <= most ? all : most > 2048 ? most : all < 2048 ? all : 2048;
    }
    p.fixed = p.keep && a->type == STBPE_REAL_BF16 && p.rows * a->vocab * 2 > FIXED_BYTES;
    p.group = group_of(p.chunk_rows < p.rows ? p.chunk_rows : p.rows, a->vocab, 0, 0, a->dim, 0, false, false);
    p.parts = (int)((a->vocab + 64 * p.group - 1) / (64 * p.group));
    p.part_stride = p.chunk_rows;
    p.few = !p.want_grads && !p.k && aligned && p.rows > 0 && p.rows <= FEW_ROWS && p.dim * (p.rows <= 2 ? p.rows : p.rows <= 4 ? 4 : 8) <= FEW_NUMBERS;
    if (p.few) p.parts = (int)(a->vocab < 8 * 4 * 2 * SMS ? (a->vocab + 31) / 32 : 2 * SMS), p.part_stride = FEW_ROWS;
    p.acc_stride = up_to(a->dim, 32);
    bytes = 0;
    char *base = (char *)a->workspace;
    auto take = [&](i64 n) {
        char *at = base + bytes;
        bytes += up_to(n, 1024);
        return (void *)at;
    };
    p.meta = (Meta *)take(sizeof(Meta));
    p.row_of = (int *)take(p.rows_padded * 4);
    p.slot_of = (int *)take(p.rows_padded * 4);
    p.plogp = (float *)take(p.rows_padded * 4);
    p.entries = (int2 *)take(p.rows_padded * 8 * (p.k ? p.k : 1));
    if (p.k) {
        p.first = (unsigned short *)take(p.rows_padded * 2 * p.pieces);
        p.has_entries = (unsigned char *)take(p.rows_padded);
    }
    p.packed = take(p.rows_padded * p.dim_padded * 2);
    p.weight_rows = aligned ? a->weight : take(p.vocab * p.dim_padded * 2);
    if (!p.lse2) p.lse2 = (float *)take(p.rows_padded * 4);
    if (p.want_loss) {
        p.entry_z = (float *)take(p.rows_padded * 4 * (p.k ? p.k : 1));
        p.part_max = (float *)take(p.part_stride * 4 * p.parts);
        p.part_sum = (float *)take(p.part_stride * 4 * p.parts);
        p.row_loss = a->reduction == STBPE_REDUCE_NONE ? a->loss : (float *)take(p.rows_padded * 4);
    }
    if (p.want_grads) {
        p.coef = (float *)take(p.rows_padded * 4);
        p.g = take(p.chunk_rows * p.g_stride * 2);
        p.split_sums = (float *)take((i64)2 * SMS * 8 * 64 * 2 * 32 * 4);
        p.split_done = (unsigned int *)take(2 * SMS * 8 * 4);
        if (!p.keep && refines(p)) p.refined = (int2 *)take(p.rows_padded * 8);
        if (p.fixed) {
            p.reference = (float *)take(p.rows_padded * 4);
            p.out_row = (float *)take(p.rows_padded * 4);
            p.again = (int *)take(2 * p.rows_padded / TILE_ROWS * 4);
            p.scaled = take(p.chunk_rows * p.dim_padded * 2);
        }
        if (p.chunk_rows < p.rows_padded && p.grad_weight) p.weight_acc = (float *)take(p.vocab * p.acc_stride * 4);
        if (p.g_stride < all && p.grad_hidden) p.acc = (float *)take(p.rows_padded * p.acc_stride * 4);
    }
    return STBPE_OK;
}

// A matrix of 16-bit numbers for TMA: boxes of 64 columns (128 bytes, swizzled) by `box` rows, zeros outside.
int tensor_map(CUtensorMap *map, int type, const void *at, i64 rows, i64 cols, i64 stride, int box, char *err, size_t err_len) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    if (!encode) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        VCK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !f) return fail(err, err_len, STBPE_E_CUDA, "cuTensorMapEncodeTiled", "not found");
        encode = (Encode)f;
    }
    const cuuint64_t size[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, pitch[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t tile[2] = {64, (cuuint32_t)box}, one[2] = {1, 1};
    const CUresult r = encode(map, type == STBPE_REAL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                              const_cast<void *>(at), size, pitch, tile, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? STBPE_OK : fail(err, err_len, STBPE_E_CUDA, "cuTensorMapEncodeTiled", "refused");
}

// launched while the kernel before still runs (next_may_come, before_is_done)
template <class... P, class... A>
cudaError_t start(void (*kernel)(P...), i64 blocks, int threads, size_t smem, int group, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)blocks), c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem, c.stream = s;
    cudaLaunchAttribute how[2];
    how[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    how[0].val.programmaticStreamSerializationAllowed = 1;
    how[1].id = cudaLaunchAttributeClusterDimension;
    how[1].val.clusterDim = {(unsigned)group, 1, 1};
    c.attrs = how, c.numAttrs = group > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

template <class T, int KIND, int GROUP>
int launch(const Plan &p, const Job &job, const Maps &maps, i64 tiles, cudaStream_t s, char *err, size_t err_len) {
    auto *kernel = product_kernel<T, KIND, GROUP>;
    VCK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PRODUCT_SMEM));
    VCK(start(kernel, (tiles < SMS / GROUP ? tiles : SMS / GROUP) * GROUP, PRODUCT_THREADS, PRODUCT_SMEM, GROUP, s, p, job, maps));
    return STBPE_OK;
}

template <class T, int KIND>
int product(const Plan &p, const Job &job, const Maps &maps, cudaStream_t s, char *err, size_t err_len) {
    const i64 rows = p.rows < job.rows ? p.rows : job.rows;
    if (KIND != GRADS) {
        if (rows == 0) return STBPE_OK;
        const i64 side = 128 * p.group, tiles = ((rows + side - 1) / side) * ((job.width + side - 1) / side);
        return p.group == 1 ? launch<T, KIND, 1>(p, job, maps, tiles, s, err, err_len) : launch<T, KIND, 2>(p, job, maps, tiles, s, err, err_len);
    }
    const i64 tall = p.grad_hidden ? rows : 0, wide = p.grad_weight ? job.width : 0;
    auto work = [&](i64 x, i64 deep) { return ((x + 255) / 256) * ((p.dim + 255) / 256) * ((deep + 63) / 64); };
    if (tall && wide && work(tall, job.width) + work(wide, rows) > 1000 * SMS / 2) {  // above 1000 steps of a cluster, 0.4 ms, a launch each
        Plan one = p;
        one.grad_weight = nullptr;
        VTRY((product<T, KIND>(one, job, maps, s, err, err_len)));
        one.grad_weight = p.grad_weight, one.grad_hidden = nullptr;
        Job rest = job;
        rest.add_up = false;
        return product<T, KIND>(one, rest, maps, s, err, err_len);
    }
    const int group = group_of(tall, p.dim, wide, p.dim, job.width, rows, !p.acc, !p.weight_acc);
    return group == 1 ? launch<T, KIND, 1>(p, job, maps, SMS, s, err, err_len) : launch<T, KIND, 2>(p, job, maps, SMS, s, err, err_len);
}

template <class T>
int run(const Plan &p, int type, cudaStream_t s, char *err, size_t err_len) {
    const int wide = SMS * 8;
    auto blocks = [&](i64 n, i64 per) { return (unsigned)(n <= 0 ? 1 : (n + per - 1) / per < wide ? (n + per - 1) / per : wide); };
    auto map = [&](CUtensorMap *m, const void *at, i64 rows, i64 cols, i64 stride, int box) {
        return tensor_map(m, type, at, rows, cols, stride, box, err, err_len);
    };
    if (p.few) {
        auto *few = p.rows == 1 ? few_kernel<T, 1> : p.rows == 2 ? few_kernel<T, 2> : p.rows <= 4 ? few_kernel<T, 4> : few_kernel<T, 8>;
        VCK(start(few, p.parts, 256, 0, 1, s, p));
        VCK(start(join_kernel<T>, 1, 256, 0, 1, s, p, 0, p.rows_padded, 1, 1));
        return STBPE_OK;
    }
    if (p.k) {
        auto *teacher = p.k <= 32 ? teacher_kernel<1> : p.k <= 64 ? teacher_kernel<2> : p.k <= 128 ? teacher_kernel<4> : teacher_kernel<8>;
        VCK(start(teacher, blocks(p.rows, 4), 128, 0, 1, s, p));
    }
    VCK(start(rows_kernel<T>, p.weight_rows != p.weight ? SMS : p.row_blocks, 1024, 0, 1, s, p));
    Maps logits, grads;
    VTRY(map(&logits.map[0], p.packed, p.rows_padded, p.dim, p.dim_padded, 128));
    VTRY(map(&logits.map[1], p.weight_rows, p.vocab, p.dim, p.weight_rows_stride, 128));
    logits.map[2] = logits.map[3] = logits.map[0];
    if (p.want_grads) {
        VTRY(map(&grads.map[0], p.g, p.chunk_rows, p.g_stride, p.g_stride, 128));
        VTRY(map(&grads.map[1], p.weight_rows, p.vocab, p.dim, p.weight_rows_stride, 64));
        VTRY(map(&grads.map[2], p.g, p.chunk_rows, p.g_stride, p.g_stride, 64));
        VTRY(map(&grads.map[3], p.fixed ? p.scaled : p.packed, p.fixed ? p.chunk_rows : p.rows_padded, p.dim, p.dim_padded, 64));
    }
    const unsigned joins = blocks(p.chunk_rows < p.rows ? p.chunk_rows : p.rows, 8);
    const int slices = p.keep && !p.fixed && joins <= SMS / 2 ? 8 : 1;  // (two slices of 1 665 rows cost 8 us, eight of 256 save 4)
    if (p.keep) {
        for (i64 r0 = 0; r0 < p.rows_padded; r0 += p.chunk_rows) {
            Job job{0, p.vocab, r0, p.chunk_rows, false, false};
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                if (p.fixed) VTRY((product<T, MAKE_E>(p, job, logits, s, err, err_len)));
            }
            if (!p.fixed) VTRY((product<T, MAKE_R>(p, job, logits, s, err, err_len)));
            VCK(start(join_kernel<T>, joins * slices, 256, 0, 1, s, p, r0, p.chunk_rows, slices, 0));
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                job.again = true;
                if (p.fixed) VTRY((product<T, MAKE_E>(p, job, logits, s, err, err_len)));
                job.again = false;
            }
            job.add_up = p.reduction != STBPE_REDUCE_NONE && r0 + p.chunk_rows >= p.rows_padded;
            VTRY((product<T, GRADS>(p, job, grads, s, err, err_len)));
        }
    } else {
        if (p.want_loss) {
            const i64 chunks = (p.rows_padded + p.chunk_rows - 1) / p.chunk_rows;
            for (i64 r0 = 0; r0 < p.rows_padded; r0 += p.chunk_rows) {
                VTRY((product<T, STATS>(p, Job{0, p.vocab, r0, p.chunk_rows, false, false}, logits, s, err, err_len)));
                VCK(start(join_kernel<T>, joins, 256, 0, 1, s, p, r0, p.chunk_rows, 1, joins * chunks));
            }
        }
        if (p.want_grads) {
            if (p.refined) VCK(start(refine_kernel<T>, blocks(p.rows, 8), 256, 0, 1, s, p));
            for (i64 v0 = 0; v0 < p.vocab; v0 += p.g_stride) {
                const Job job{v0, p.vocab - v0 < p.g_stride ? p.vocab - v0 : p.g_stride, 0, p.rows_padded, false, false};
                VTRY((product<T, MAKE_G>(p, job, logits, s, err, err_len)));
                VTRY((product<T, GRADS>(p, job, grads, s, err, err_len)));
            }
            if (p.grad_hidden && p.acc) VCK(start(scatter_kernel<T>, blocks(p.rows * p.dim, 256), 256, 0, 1, s, p));
        }
    }
    return STBPE_OK;
}

}  // namespace

extern "C" {

STBPE_VISIBLE int stbpe_vocab_loss_workspace(const stbpe_vocab_loss *args, int64_t *bytes, char *err, size_t err_len) {
    Plan p;
    i64 need = 0;
    if (err && err_len) err[0] = 0;
    const int st = plan(args, p, need, err, err_len);
    if (st == STBPE_OK && bytes) *bytes = need;
    return st;
}

STBPE_VISIBLE int stbpe_scale_gradients(void *a, int64_t n_a, void *b, int64_t n_b, const float *by, void *stream) {
    if (n_a < 0 || n_b < 0 || (n_a && !a) || (n_b && !b) || !by || (uintptr_t)a % 16 || (uintptr_t)b % 16) return STBPE_E_BADARG;
    const i64 most = n_a > n_b ? n_a : n_b;
    if (most == 0) return STBPE_OK;
    const i64 blocks = (most + 2047) / 2048;
    if (start(scale_kernel, blocks < SMS * 8 ? blocks : SMS * 8, 256, 0, 1, (cudaStream_t)stream, (__nv_bfloat16 *)a, n_a, (__nv_bfloat16 *)b,
              n_b, by) == cudaSuccess)
        return STBPE_OK;
    cudaGetLastError();
    return STBPE_E_CUDA;
}

STBPE_VISIBLE int stbpe_vocab_loss_run(const stbpe_vocab_loss *args, void *stream, char *err, size_t err_len) {
    Plan p;
    i64 need = 0;
    if (err && err_len) err[0] = 0;
    const int st = plan(args, p, need, err, err_len);
    if (st != STBPE_OK) return st;
    if (!args->workspace || (uintptr_t)args->workspace % 1024 || args->workspace_bytes < need)
        return fail(err, err_len, STBPE_E_CAPACITY, "stbpe_vocab_loss", "workspace missing, not on a 1024-byte boundary or too small");
    if ((!p.want_loss && !args->lse2) || (p.want_loss && !args->loss) || (p.want_grads && p.rows && !args->grad_hidden && !args->grad_weight))
        return fail(err, err_len, STBPE_E_BADARG, "stbpe_vocab_loss", "an output is missing");
    if ((uintptr_t)args->grad_hidden % 16 || (uintptr_t)args->grad_weight % 16)
        return fail(err, err_len, STBPE_E_BADARG, "stbpe_vocab_loss", "gradients start on 16-byte boundaries");
    if (!args->weight || (p.rows && (!args->hidden || !args->ids || (p.k && !args->logits))))
        return fail(err, err_len, STBPE_E_BADARG, "stbpe_vocab_loss", "an input is missing");
    return args->type == STBPE_REAL_BF16 ? run<__nv_bfloat16>(p, args->type, (cudaStream_t)stream, err, err_len)
                                         : run<__half>(p, args->type, (cudaStream_t)stream, err, err_len);
}

}  // extern "C"
