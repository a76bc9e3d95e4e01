// The products of the losses over a large vocabulary on the tensor cores: tcgen05 with its operands in shared memory, filled by
// TMA, and its sums (32 bits) in TMEM.
//
//   STATS        Z = H W^T; per row and part of the columns the maximum and the sum of exp, the logits at the entries
//   MAKE_E       the same, and E = exp2(Z - reference) in 16 bits
//   MAKE_R       the same with each part's maximum, less 14, as the reference: E is below 2^14
//   MAKE_G       Z again, of one piece of the vocabulary, and G = dlogits from it in 16 bits
//   GRADS        dH = E W or G W        (k over the columns: W is read with the other dimension contiguous) and
//                dW = E^T H' or G^T H   (k over the rows: both are read with the other dimension contiguous),
//                which wait for the same and fill each other's last round: a step over 2 048 x 1 256 x 512 took 42 us with
//                both in one launch and 51 with one each
//
// A group of GROUP CTAs makes a tile of 128 GROUP x 128 GROUP: with GROUP = 2 the two CTAs of a cluster share one
// 256 x 256 tile (cta_group::2), each holding its half of both operands, so that a byte brought into shared memory serves twice as
// many products.  A CTA loads 128 x 64 of each operand per step in either case: 64 bytes per SM and clock at the full rate
// with GROUP = 2, 128 with GROUP = 1, which L2 does not deliver (1.5 to 1.6 PFLOP/s against 0.93 to 0.98 at
// 8 188 x 32 256 x 2 048).  Persistent: the tiles are dealt out to the clusters in turn, and the sums of one tile are looked at
// while the next one is being made (two buffers in TMEM).
// Warp 0 loads, warp 1 of the group's first CTA multiplies, warp 2 owns the TMEM, warps 4 to 11 take the sums, warp 3 has
// the losses to add up.
//
// What bounds them at that size: the tensor pipe, active 92 to 95 % of the cycles, and the board's power, which holds the clock at
// 1.35 to 1.45 GHz.  At depths of 12 steps or fewer the instructions and latencies of the exponentials, two warps to a scheduler (4 500 x
// 32 494 x 128 scored in 107 us, of which the exponentials' pipe is busy 41); where the tiles are few, what begins and ends one.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "vocab_loss.cuh"

namespace vloss {

enum { STATS, MAKE_E, MAKE_R, MAKE_G, GRADS };

constexpr int STAGES = 6;
constexpr int OPERAND_BYTES = 128 * 64 * 2;  // what a CTA loads of one operand per step of 64 terms
constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
constexpr int SPLITS = 8;
constexpr int PRODUCT_THREADS = 384;
constexpr int PRODUCT_SMEM = STAGES * STAGE_BYTES + 1024 + 256 + 8 * 2048;

// How the tiles of one or two results are dealt out: whole ones in rounds of all clusters, and those that are left behind a result's full
// rounds split in depth, up to SPLITS units per tile of SPLIT_STEPS steps at least, so that the last round is shorter, too.  Joining
// a units of a tile costs about as much as JOIN_STEPS + 2 a steps.
constexpr int SPLIT_STEPS = 16, JOIN_STEPS = 8;
struct Deal {
    unsigned whole[2], left[2], splits[2], units;
    unsigned steps;  // what the busiest cluster goes through, about
};
__host__ __device__ inline Deal deal(const unsigned (&tiles)[2], const unsigned (&steps)[2], const bool (&may_split)[2], unsigned clusters) {
    Deal d;
    unsigned rounds = 0, most[2];
    for (int r = 0; r < 2; ++r) {
        d.left[r] = tiles[r] % clusters, d.whole[r] = tiles[r] - d.left[r], d.splits[r] = 1;
        rounds += d.whole[r] / clusters * steps[r];
        most[r] = may_split[r] && d.left[r] ? SPLITS : 1;
        while (most[r] > 1 && (steps[r] < most[r] * SPLIT_STEPS || d.left[r] * most[r] > clusters)) most[r] >>= 1;
    }
    unsigned best = UINT_MAX;
    for (unsigned a = 1; a <= most[0]; a *= 2)
        for (unsigned b = 1; b <= most[1]; b *= 2) {
            const unsigned x = d.left[0] ? steps[0] / a + (a > 1 ? JOIN_STEPS + 2 * a : 0) : 0;
            const unsigned y = d.left[1] ? steps[1] / b + (b > 1 ? JOIN_STEPS + 2 * b : 0) : 0;
            const unsigned cost = d.left[0] * a + d.left[1] * b <= clusters ? (x > y ? x : y) : x + y;
            if (cost < best) best = cost, d.splits[0] = a, d.splits[1] = b;
        }
    d.units = d.whole[0] + d.whole[1] + d.left[0] * d.splits[0] + d.left[1] * d.splits[1];
    d.steps = rounds + best;
    return d;
}

struct Maps {
    CUtensorMap map[4];
};

struct Job {
    i64 v0, width;  // the piece of the vocabulary
    i64 r0, rows;   // the chunk of the packed rows
    bool again;     // MAKE_E: only where a reference was too far off
    bool add_up;    // GRADS: the losses are added up beside the products
};

// ---------------------------------------------------------------------------------------------- instructions
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// nothing in memory goes with it (the loads from TMEM have arrived), so it does not wait for the thread's stores
__device__ __forceinline__ void barrier_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Every wait ends: after two seconds it fails, all roles leave their loops as that happens to them, and what was to be
// computed becomes NaN.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    u64 began = 0;
    for (;;) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity), "r"(100000)  // ns that the hardware may sleep at a time
            : "memory");
        if (done) return true;
        u64 now;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (!began) began = now;
        if (now - began > 2000000000ull) return false;
    }
}

template <int GROUP>
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if (GROUP == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map),
            "r"(x), "r"(y), "r"(bar)
            : "memory");
}

template <int GROUP>
__device__ __forceinline__ void mma(uint32_t tmem, u64 a, u64 b, uint32_t what, uint32_t add) {
    if (GROUP == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(what), "r"(add)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                     "l"(a), "l"(b), "r"(what), "r"(add)
                     : "memory");
}

// arrives at the barrier (of both CTAs of a pair) when the products issued so far are done
template <int GROUP>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if (GROUP == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((unsigned short)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(at)
        : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two numbers by one instruction
__device__ __forceinline__ u64 two(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void fma_two(float &a, float &b, u64 times, u64 plus) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(two(a, b)), "l"(times), "l"(plus));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ u64 add_two(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// (NaN is left out, as by fmaxf)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// the largest of N, in four chains of operations side by side
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
    float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int x = 4; x < N; x += 8)
#pragma unroll
        for (int y = 0; y < 4; ++y) m[y] = x + 4 + y < N ? max3(m[y], v[x + y], v[x + 4 + y]) : fmaxf(m[y], v[x + y]);
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Descriptor of an operand in shared memory, 128-byte swizzle.  Contiguous along k: rows of 128 bytes, eight rows to the
// next at 1024 (the other offset is unused).  Contiguous along the other dimension: slabs of 64 of them by 64 k, eight k to
// the next at 1024, the next slab at 8192.
template <bool ALONG_K>
__device__ __forceinline__ u64 operand(uint32_t addr) {
    const u64 leading = ALONG_K ? 1 : 8192 >> 4, stride = 1024 >> 4;
    return (u64)((addr & 0x3FFFF) >> 4) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(uint32_t *)&v;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *(uint32_t *)&v;
}

// 32 columns of a warp's 32 rows in 16 bits, a row to a lane, by way of shared memory (2 KB of the warp's own), so that lanes side by side
// store to one row: 16 bytes by 4 lanes, 4 by 16 or 2 by 32 (`unit` numbers at a time), where a lane that stores its own row
// touches a sector of its own each time.  `to`: where the lane's row goes, null: nowhere; `inside`: how many of the columns there are.
template <class T, int N>
__device__ __forceinline__ void store_rows(T *to, const float (&w)[N], i64 inside, int unit, uint32_t stage, int lane) {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c)  // units of 16 bytes change places so that eight rows fall into different banks
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + (c ^ ((lane >> 1) & 3)) * 16),
                     "r"(pack2<T>(w[8 * c], w[8 * c + 1])), "r"(pack2<T>(w[8 * c + 2], w[8 * c + 3])),
                     "r"(pack2<T>(w[8 * c + 4], w[8 * c + 5])), "r"(pack2<T>(w[8 * c + 6], w[8 * c + 7]))
                     : "memory");
    __syncwarp();
    if (unit == 8 && inside >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), c = lane & 3;
            uint4 x;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                         : "r"(stage + row * 64 + (c ^ ((row >> 1) & 3)) * 16)
                         : "memory");
            T *at = (T *)__shfl_sync(~0u, (u64)to, row);
            if (at) *(uint4 *)(at + c * 8) = x;
        }
    } else if (unit >= 2 && inside >= 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = i * 2 + (lane >> 4), c = (lane & 15) >> 2;
            uint32_t x;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(stage + row * 64 + (c ^ ((row >> 1) & 3)) * 16 + (lane & 3) * 4) : "memory");
            T *at = (T *)__shfl_sync(~0u, (u64)to, row);
            if (at) *(uint32_t *)(at + (lane & 15) * 2) = x;
        }
    } else {
#pragma unroll 8
        for (int row = 0; row < 32; ++row) {
            unsigned short x;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(stage + row * 64 + ((lane >> 3) ^ ((row >> 1) & 3)) * 16 + (lane & 7) * 2) : "memory");
            T *at = (T *)__shfl_sync(~0u, (u64)to, row);
            if (at && lane < inside) *(unsigned short *)(at + lane) = x;
        }
    }
}

// The entries of one row in ascending order: what falls into the columns at hand.  The one behind the next is on its way already.
struct Walk {
    const int2 *entries;
    int at, all;
    int2 next, then;

    __device__ __forceinline__ int2 entry(int which) const { return which < all ? entries[which] : make_int2(INT_MAX, 0); }
    __device__ __forceinline__ void start(const Plan &p, i64 row, i64 column) {
        all = p.k ? p.k : 1;
        entries = p.entries + row * all;
        at = p.k ? p.first[row * p.pieces + column / PIECE] : 0;
        next = entry(at), then = entry(at + 1);
        while (next.x < column) advance();
    }
    __device__ __forceinline__ void advance() {
        ++at;
        next = then;
        then = entry(at + 1);
    }
};

// ---------------------------------------------------------------------------------------------- the kernel
// maps: H and W (logits); E or G and W for dH, E or G and H for dW
template <class T, int KIND, int GROUP>
__global__ void __launch_bounds__(PRODUCT_THREADS, 1)
    product_kernel(const __grid_constant__ Plan p, const __grid_constant__ Job job, const __grid_constant__ Maps maps) {
    constexpr bool LOGITS = KIND != GRADS;
    constexpr int TILE = 128 * GROUP, COLUMNS = TILE / 2;  // columns that one epilogue thread takes of its row,
    constexpr int W = KIND == STATS ? 64 : 32;             // and how many at a time
    // sums in 32 bits, the operands' type, TILE x TILE; dH has only its second operand across, dW both
    constexpr uint32_t WHAT = 1u << 4 | (std::is_same<T, __nv_bfloat16>::value ? 1u << 7 | 1u << 10 : 0u) | (LOGITS ? 0u : 1u << 16) |
                              (uint32_t)(TILE >> 3) << 17 | (uint32_t)(TILE >> 4) << 24;
    constexpr uint32_t A_ACROSS = 1u << 15;
    extern __shared__ char raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t bars = base + STAGES * STAGE_BYTES;
    const uint32_t full = bars, empty = bars + 8 * STAGES, sums_full = bars + 16 * STAGES, sums_empty = sums_full + 16,
                   drained = sums_full + 32, tmem_at = sums_full + 40;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank = 0;
    if (GROUP == 2) asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));

    next_may_come();
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < STAGES; ++s) barrier_init(full + 8 * s, 1), barrier_init(empty + 8 * s, 1);
        for (int b = 0; b < 2; ++b) barrier_init(sums_full + 8 * b, 1), barrier_init(sums_empty + 8 * b, 8 * GROUP);
        barrier_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
#pragma unroll
        for (int x = 0; x < (LOGITS ? 2 : 4); ++x) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.map[x]) : "memory");
    }
    if (warp == 2) {
        if (GROUP == 2)
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_at), "r"(2 * TILE) : "memory");
        else
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_at), "r"(2 * TILE) : "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncthreads();
    if (GROUP == 2) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));

    before_is_done();
    // The tiles and their depth.  Result 0 is Z or dH, result 1 is dW.
    const i64 counted = p.meta->counted;
    const i64 n = counted - job.r0 < 0 ? 0 : counted - job.r0 < job.rows ? counted - job.r0 : job.rows;  // rows of this chunk
    const unsigned cluster = blockIdx.x / GROUP, clusters = gridDim.x / GROUP;
    const i64 rows[2] = {n, job.width}, cols[2] = {LOGITS ? job.width : p.dim, p.dim};
    const unsigned steps[2] = {(unsigned)(((LOGITS ? p.dim : job.width) + 63) / 64), (unsigned)((n + 63) / 64)};
    unsigned tiles_m[2], tiles_n[2], tiles[2], band[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        tiles_m[r] = (unsigned)((rows[r] + TILE - 1) / TILE), tiles_n[r] = (unsigned)((cols[r] + TILE - 1) / TILE);
        tiles[r] = tiles_m[r] * tiles_n[r];
        // A band of tiles of rows goes through all columns, its rows first.  Z: that much of H stays in L2 while W passes by.  Else the
        // tiles that are being made at a time are as many columns as there are, or a square where both operands pass by, so that
        // they share what comes from memory.
        band[r] = LOGITS ? 16 : (clusters + tiles_n[r] - 1) / tiles_n[r];
        if (!LOGITS && r == 0 && band[r] < 16 / GROUP) band[r] = 16 / GROUP;
    }
    if (LOGITS || !p.grad_weight || (job.r0 > 0 && n == 0)) tiles[1] = 0;
    if ((!LOGITS && !p.grad_hidden) || (KIND == MAKE_E && job.again && !p.meta->again)) tiles[0] = 0;
    const Deal dealt = deal(tiles, steps, {!LOGITS && !p.acc, !LOGITS && !p.weight_acc}, clusters);
    const unsigned units = dealt.units;
    struct Unit {
        i64 m0, n0;
        int k0, k1, split, splits;  // steps; split < 0: the whole tile
        int result, sums, done;     // where its sums go and are counted, if it is split
    };
    auto unit_at = [&](unsigned u) {  // (32-bit divisions: this stands between two tiles)
        Unit t;
        // dH, whose tiles go deeper as a rule, and what is left of it, then dW
        const unsigned first = dealt.left[0] * dealt.splits[0];
        t.result = u >= dealt.whole[0] + first;
        unsigned x = t.result ? u - dealt.whole[0] - first : u, tile = x;
        const unsigned whole = t.result ? dealt.whole[1] : dealt.whole[0], left = t.result ? dealt.left[1] : dealt.left[0];
        t.split = -1, t.splits = 1, t.sums = t.done = 0;
        if (x >= whole) {
            x -= whole;
            const unsigned split = x / left, index = x - split * left;
            tile = whole + index;
            t.splits = (int)(t.result ? dealt.splits[1] : dealt.splits[0]);
            if (t.splits > 1) {
                t.split = (int)split;
                t.sums = (int)((t.result ? first : 0) + index * t.splits), t.done = (int)((t.result ? dealt.left[0] : 0) + index);
            }
        }
        const unsigned deep = t.result ? steps[1] : steps[0], high_m = t.result ? tiles_m[1] : tiles_m[0],
                       wide_n = t.result ? tiles_n[1] : tiles_n[0], b = t.result ? band[1] : band[0];
        t.k0 = t.split < 0 ? 0 : (int)(deep * (unsigned)t.split / (unsigned)t.splits);
        t.k1 = t.split < 0 ? (int)deep : (int)(deep * (unsigned)(t.split + 1) / (unsigned)t.splits);
        const unsigned which = tile / (b * wide_n), in = tile - which * b * wide_n;
        const unsigned high = high_m - which * b < b ? high_m - which * b : b, column = in / high;
        t.n0 = (i64)column * TILE;
        t.m0 = (i64)(which * b + in - column * high) * TILE;
        return t;
    };
    auto skipped = [&](const Unit &t) { return KIND == MAKE_E && job.again && !p.again[(job.r0 + t.m0) / TILE_ROWS]; };

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 0;
            i64 issued = 0;
            bool alive = true;
            for (unsigned u = cluster; u < units && alive; u += clusters) {
                const Unit t = unit_at(u);
                if (skipped(t)) continue;
                const int am = (int)(t.m0 + rank * 128), bn = (int)(t.n0 + rank * 128), h0 = p.fixed ? 0 : (int)job.r0;
                // (a loop of its own for each result: what differs is known when it is compiled)
                auto load = [&](auto which) {
                    constexpr int RESULT = decltype(which)::value;
                    for (int k = t.k0; k < t.k1; ++k) {
                        if (!barrier_wait(empty + 8 * s, phase ^ 1)) {
                            alive = false;
                            break;
                        }
                        const uint32_t a = base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
                        const uint32_t bar = GROUP == 2 ? in_cta(full + 8 * s, 0) : full + 8 * s;
                        if (rank == 0) barrier_expect(full + 8 * s, GROUP * STAGE_BYTES);
                        if (LOGITS) {
                            tma_load<GROUP>(a, &maps.map[0], k * 64, (int)job.r0 + am, bar);
                            tma_load<GROUP>(b, &maps.map[1], k * 64, (int)job.v0 + bn, bar);
                        } else if (RESULT == 0) {
                            tma_load<GROUP>(a, &maps.map[0], k * 64, am, bar);
                            tma_load<GROUP>(b, &maps.map[1], bn, (int)job.v0 + k * 64, bar);
                            tma_load<GROUP>(b + 8192, &maps.map[1], bn + 64, (int)job.v0 + k * 64, bar);
                        } else {
                            tma_load<GROUP>(a, &maps.map[2], am, k * 64, bar);
                            tma_load<GROUP>(a + 8192, &maps.map[2], am + 64, k * 64, bar);
                            tma_load<GROUP>(b, &maps.map[3], bn, h0 + k * 64, bar);
                            tma_load<GROUP>(b + 8192, &maps.map[3], bn + 64, h0 + k * 64, bar);
                        }
                        ++issued;
                        if (++s == STAGES) s = 0, phase ^= 1;
                    }
                };
                if (LOGITS || t.result == 0) load(std::integral_constant<int, 0>());
                else load(std::integral_constant<int, 1>());
            }
            if (!alive && rank == 0) {  // copies in flight land before the memory is given up
                const i64 pending = issued < STAGES ? issued : STAGES;
                for (i64 x = issued - pending; x < issued; ++x) barrier_wait(full + 8 * (int)(x % STAGES), (uint32_t)(x / STAGES & 1));
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int s = 0, buffer = 0;
            uint32_t phase = 0, sums_phase = 0;
            bool alive = true;
            for (unsigned u = cluster; u < units && alive; u += clusters) {
                const Unit t = unit_at(u);
                if (skipped(t)) continue;
                if (!barrier_wait(sums_empty + 8 * buffer, sums_phase ^ 1)) {
                    alive = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + buffer * TILE;
                auto multiply = [&](auto which) {
                    constexpr int RESULT = decltype(which)::value;
                    constexpr u64 ALONG = 32 >> 4, ACROSS = 2048 >> 4;  // 16 k further
                    for (int k = t.k0; k < t.k1; ++k) {
                        if (!barrier_wait(full + 8 * s, phase)) {
                            alive = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const u64 a = operand<RESULT == 0>(base + s * STAGE_BYTES), b = operand<LOGITS>(base + s * STAGE_BYTES + OPERAND_BYTES);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            mma<GROUP>(d, a + x * (RESULT == 0 ? ALONG : ACROSS), b + x * (LOGITS ? ALONG : ACROSS), RESULT == 0 ? WHAT : WHAT | A_ACROSS,
                                       k > t.k0 || x > 0);
                        mma_commit<GROUP>(empty + 8 * s);
                        if (++s == STAGES) s = 0, phase ^= 1;
                    }
                };
                if (LOGITS || t.result == 0) multiply(std::integral_constant<int, 0>());
                else multiply(std::integral_constant<int, 1>());
                if (alive) mma_commit<GROUP>(sums_full + 8 * buffer);
                buffer ^= 1;
                if (buffer == 0) sums_phase ^= 1;
            }
            if (!alive) {  // products in flight end before the TMEM is given up
                mma_commit<GROUP>(drained);
                barrier_wait(drained, 0);
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        if (!LOGITS && job.add_up && blockIdx.x == 0) add_up(p, lane);
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const float scale = p.inv_temperature * 1.4426950408889634f;
        const int entries_of_row = p.k ? p.k : 1;
        const uint32_t stage = bars + 256 + (warp - 4) * 2048;
        const int unit = p.dim % 8 == 0 ? 8 : p.dim % 2 == 0 ? 2 : 1;  // of the caller's rows
        int buffer = 0;
        uint32_t sums_phase = 0;
        bool alive = true;  // once a wait has run out, all that is left becomes NaN
        for (unsigned u = cluster; u < units; u += clusters) {
            const Unit t = unit_at(u);
            if (skipped(t)) continue;
            const i64 m = t.m0 + rank * 128 + quarter * 32 + lane;  // this thread's row of the result
            const i64 c0 = t.n0 + half * COLUMNS;                   // and its first column
            const i64 slot = job.r0 + m;
            int row = -1;
            // exp2(0 - inf) = 0 in the rows that fill the last tile up
            float shift = INFINITY, coef = 0.f, top = LOWEST, sum = 0.f;
            int2 refined = make_int2(-1, 0);
            Walk walk;
            if (LOGITS) {
                row = slot < p.rows_padded ? p.row_of[slot] : -1;
                if (row >= 0 && job.v0 + c0 < p.vocab) walk.start(p, row, job.v0 + c0);
                else walk.next.x = walk.then.x = INT_MAX, walk.at = walk.all = 0;
                if (KIND == MAKE_E && row >= 0) shift = p.reference[slot];
                if (KIND == MAKE_G && row >= 0) {
                    shift = p.lse2[row], coef = p.coef[slot] * p.meta->in_scale;
                    if (p.refined) refined = p.refined[slot];
                }
            }
            // E and G of the rows that fill the last tile up are 0 whatever the weight holds (0 times a weight of -inf is NaN)
            const bool filled = LOGITS && KIND != STATS && __any_sync(~0u, row < 0);
            if (!LOGITS) {
                coef = p.meta->out_scale;
                if (t.result == 0 && m < n) {
                    row = p.row_of[slot];
                    if (p.fixed) coef = p.out_row[slot];
                }
            }
            // 32 sums of dH or dW, at column c of this thread's columns
            auto emit = [&](int c, float(&v)[32]) {
                if (c0 + c >= p.dim) return;
                if (t.result == 0) {
                    if (!p.acc) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] *= coef;
                        store_rows(m < n ? (T *)p.grad_hidden + (i64)row * p.dim + c0 + c : nullptr, v, p.dim - c0 - c, unit, stage, lane);
                    } else if (m < n) {
                        float4 *to = (float4 *)(p.acc + m * p.acc_stride + c0 + c);
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            float4 y = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
                            if (job.v0 > 0) {
                                const float4 z = to[x];
                                y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                            }
                            to[x] = y;
                        }
                    }
                } else {
                    const i64 id = job.v0 + m;
                    const bool there = m < job.width, last = counted <= job.r0 + job.rows;
                    float4 *to = (float4 *)(p.weight_acc + id * p.acc_stride + c0 + c);
                    if (job.r0 > 0 && there) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const float4 z = to[x];
                            v[4 * x] += z.x, v[4 * x + 1] += z.y, v[4 * x + 2] += z.z, v[4 * x + 3] += z.w;
                        }
                    }
                    if (last) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] *= coef;
                        store_rows(there ? (T *)p.grad_weight + id * p.dim + c0 + c : nullptr, v, p.dim - c0 - c, unit, stage, lane);
                    } else if (there) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) to[x] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
                    }
                }
            };
            if (alive) alive = __all_sync(~0u, barrier_wait(sums_full + 8 * buffer, sums_phase));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem + buffer * TILE + half * COLUMNS + ((uint32_t)(quarter * 32) << 16);
            // [unit of a split tile][CTA][warp][column / 4][lane], four columns each
            float4 *sums = (float4 *)p.split_sums + (((i64)(t.sums + (t.split < 0 ? 0 : t.split)) * GROUP + rank) * 8 + warp - 4) * (COLUMNS * 8) + lane;
            if (KIND == MAKE_R) {  // the maximum first, the sums are read twice
#pragma unroll 1
                for (int c = 0; c < COLUMNS && alive; c += W) {
                    uint32_t bits[W];
                    __syncwarp();
                    tmem_load(from + c, bits);
                    const i64 inside = p.vocab - (job.v0 + c0 + c);
                    float v[W];
#pragma unroll
                    for (int x = 0; x < W; ++x) v[x] = __uint_as_float(bits[x]);
                    if (inside < W) {
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (x >= inside) v[x] = -INFINITY;
                    }
                    top = fmaxf(top, largest(v) * scale);
                }
                top -= 14.f;
                if (row >= 0) shift = top;
            }
#pragma unroll 1
            for (int c = 0; c < COLUMNS; c += W) {
                float v[W];
                __syncwarp();
                if (alive) {
                    uint32_t bits[W];
                    tmem_load(from + c, bits);
#pragma unroll
                    for (int x = 0; x < W; ++x) v[x] = LOGITS || t.k1 > t.k0 ? __uint_as_float(bits[x]) : 0.f;  // (no rows: nothing was summed)
                    if (c + W == COLUMNS) {  // the buffer is free
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) barrier_arrive_cluster(GROUP == 2 ? in_cta(sums_empty + 8 * buffer, 0) : sums_empty + 8 * buffer);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < W; ++x) v[x] = NAN;
                }
                if constexpr (!LOGITS) {
                    if (t.split < 0) {
                        emit(c, v);
                    } else {
#pragma unroll
                        for (int x = 0; x < W; x += 4) __stcg(sums + (c + x) * 8, make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]));
                    }
                    continue;
                }
                if (filled) {
#pragma unroll
                    for (int x = 0; x < W; ++x) v[x] = row < 0 ? 0.f : v[x];
                }
                const i64 j = job.v0 + c0 + c;  // first column, as a token id
                if (KIND != MAKE_G) {
                    while (walk.next.x < j + W) {
                        const int x0 = walk.next.x - (int)j;
                        float z = 0.f;
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (x == x0) z = v[x];
                        p.entry_z[slot * entries_of_row + walk.at] = z;
                        walk.advance();
                    }
                    if (j + W > p.vocab) {
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (j + x >= p.vocab) v[x] = -INFINITY;
                    }
                    if (KIND != MAKE_R) {
                        const float now = fmaxf(top, largest(v) * scale);
                        if (KIND == STATS) sum *= exp2_fast(top - now), shift = now;
                        top = now;
                    }
                }
                const u64 scales = two(scale, scale), shifts = two(-shift, -shift);
#pragma unroll
                for (int x = 0; x < W; x += 2) {
                    fma_two(v[x], v[x + 1], scales, shifts);
                    v[x] = exp2_fast(v[x]), v[x + 1] = exp2_fast(v[x + 1]);
                }
                if (KIND != MAKE_G) {
                    u64 part[2] = {two(v[0], v[1]), two(v[2], v[3])};
#pragma unroll
                    for (int x = 4; x < W; x += 2) part[x / 2 & 1] = add_two(part[x / 2 & 1], two(v[x], v[x + 1]));
                    float a, b;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(add_two(part[0], part[1])));
                    sum += a + b;
                }
                if (KIND == MAKE_G) {
                    while (walk.next.x < j + W) {
                        const int x0 = walk.next.x - (int)j;
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (x == x0) v[x] = (walk.at == refined.x ? __int_as_float(refined.y) : v[x]) - __int_as_float(walk.next.y);
                        walk.advance();
                    }
#pragma unroll
                    for (int x = 0; x < W; ++x) v[x] *= coef;
                    if (j + W > p.vocab) {
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (j + x >= p.vocab) v[x] = 0.f;
                    }
                }
                if (KIND != STATS) {
                    T *to = (T *)p.g + m * p.g_stride + c0 + c;
                    if (c0 + c < p.g_stride) store_rows(to, v, 32, 8, stage, lane);
                }
            }
            if (LOGITS && KIND != MAKE_G && row >= 0 && job.v0 + c0 < p.vocab) {
                const i64 to = (job.v0 + c0) / COLUMNS * p.part_stride + m;
                p.part_max[to] = top, p.part_sum[to] = sum;
            }
            if (KIND == MAKE_E && job.again) {
                // the warp that is through last with the parts of these rows joins them
                __threadfence();
                __syncwarp();
                const i64 m0 = t.m0 / TILE_ROWS * TILE_ROWS, high = n - m0 < TILE_ROWS ? n - m0 : TILE_ROWS;
                const int parts = (int)((high + TILE - 1) / TILE * tiles_n[0]) * GROUP * 8;
                int before = 0;
                if (lane == 0) before = atomicAdd(p.again + (p.rows_padded + job.r0 + m0) / TILE_ROWS, 1);
                if (__shfl_sync(~0u, before, 0) == parts - 1) {
                    __threadfence();
                    join_again<T>(p, job.r0, m0, n, lane);
                }
            }
            if (!LOGITS && t.split >= 0) {
                // the last of the splits to get here adds them up, in their order
                __threadfence();
                __syncwarp();
                unsigned int *done = p.split_done + (t.done * GROUP + rank) * 8 + warp - 4;
                unsigned int before = 0;
                if (lane == 0) before = atomicAdd(done, 1u);
                before = __shfl_sync(~0u, before, 0);
                if (before == t.splits - 1) {
                    __threadfence();
                    if (lane == 0) *done = 0;
                    constexpr int next = GROUP * 8 * COLUMNS * 8;
                    sums -= (i64)t.split * next;
#pragma unroll 1
                    for (int c = 0; c < COLUMNS; c += 32) {
                        float v[32];
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = 0.f;
#pragma unroll 1
                        for (int s = 0; s < t.splits; s += 2) {  // two units on their way at a time
                            float4 y[2][8];
#pragma unroll
                            for (int z = 0; z < 2; ++z)
#pragma unroll
                                for (int x = 0; x < 8; ++x)
                                    y[z][x] = s + z < t.splits ? __ldcg(sums + (s + z) * next + (c + 4 * x) * 8) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int z = 0; z < 2; ++z)
#pragma unroll
                                for (int x = 0; x < 8; ++x)
                                    v[4 * x] += y[z][x].x, v[4 * x + 1] += y[z][x].y, v[4 * x + 2] += y[z][x].z, v[4 * x + 3] += y[z][x].w;
                        }
                        emit(c, v);
                    }
                }
            }
            buffer ^= 1;
            if (buffer == 0) sums_phase ^= 1;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (GROUP == 2) cluster_sync();  // the other CTA may still arrive at this one's barriers
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 2) {
        if (GROUP == 2) {
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TILE));
        } else {
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TILE));
        }
    }
}

}  // namespace vloss
