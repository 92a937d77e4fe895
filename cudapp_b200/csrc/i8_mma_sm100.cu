// i8_mma_sm100.cu: the product of i8_gemm.cu on tcgen05 (kind::i8, 32-bit integer accumulators in TMEM), for more than a few rows.
//
// Weights are the M operand, activation rows the N operand: N follows a tile's row count in steps of 16 (32 for a pair of CTAs), so a ragged tile wastes no more than
// that, and one kernel serves an expert's three rows and a prefill's 256. Accumulators need no promotion on the way through k: a unit of work (a tile of rows, a block of
// 128 CG channels) runs its whole k into one accumulator and is drained once, while the next unit fills the other.
//
// What bounds it is shared memory: 128 columns of a 128 x 256 unit are written (48 KB) and read by four products (48 KB) at 128 bytes a clock, 750 clocks for 512 of
// tensor work; measured 0.33 us. CG = 2: two CTAs share a unit of 256 channels; each holds its half of the channels and of the rows, the products read both halves, and a
// row's bytes are written and read once for 256 channels: 0.25 us, the tensor cores' own rate (4096 x 4096 x 4096: 53 us with one CTA, 46 with two). Two blocks of
// 128 channels per CTA instead save the writes but not the reads and leave no second accumulator: 52 us. GATHER: the rows of a tile are fetched through a row map by
// four warps with 16-byte asynchronous copies (TMA's four-row gather takes 95 clocks a time: 308 us for the gate|up product of a 4096-token layer, whose rows in sorted order take 122).
// SPLIT: where units are fewer than SMs, a cluster of 2, 4 or 8 CTAs shares one: each takes its part of k, leaves its sums in its shared memory, and adds up its share of the
// rows over the cluster. Integer sums: the result is the same, whatever the split.
//
// Warps: 0 weights (TMA), 1 MMA issuer (of a pair's first CTA), 2 TMEM, 3 rows (TMA), 4 - 19 epilogue,
// GATHER 20 - 23 row copies. KPS: blocks of 128 columns in a stage of the ring. Every mbarrier wait is bounded; on expiry the kernel
// records a code in *err, lets its own copies land, frees its TMEM and returns, and later launches on the tensor do nothing.
#include <math.h>
#include "internal.h"
#include "mma_common.cuh"

namespace b200 {

constexpr uint32_t I8_EPI = 16, I8_STAGES = 12, I8_N_MAX = 256, I8_TEAM = 4;   // epilogue warps, most stages, most rows of a tile, warps that copy rows
constexpr uint32_t i8_threads(bool gather) { return 128 + 32 * I8_EPI + (gather ? 32 * I8_TEAM : 0); }
constexpr uint32_t I8_OUT_ROW = 80, I8_OUT = 16 * I8_OUT_ROW;     // an epilogue warp's 16 result rows of 32 bf16 channels; 80 bytes apart: neither side meets a bank twice
constexpr size_t I8_SMEM = 214 * 1024;                            // dynamic shared memory of every form: stages, result rows, alignment
constexpr uint32_t I8_ROOM = (uint32_t)I8_SMEM - 1024u - I8_EPI * I8_OUT;   // the stages' part

struct I8MmaArgs {
    const float *ws, *xs; uint16_t *y16; float *y32;
    const uint4 *tiles; const uint32_t *header, *xmap, *ymap;
    const int8_t *x; size_t x_stride; uint32_t x_rows;             // GATHER
    // n: channels of one matrix; tiles_most: all tiles of a dense product, the most of a plan; steps: 16 or 32 (pairs) dense rows each; n_cap: accumulator columns of a tile;
    // box: rows of one load; packed: bf16 rows of a multiple of 8 channels; lag: of a copying warp's stages, how many stay in flight behind the newest, 0 or 1;
    // split: CTAs of a unit; once: weights are read by one tile each and need not stay in L2
    // early: the units and their weights are known before the kernels ahead in the stream have completed
    // tile_rows: most rows that a tile of a plan may have; x_limit: without a map, rows of x (a tile's rows from there on are left out), else no limit
    uint32_t m, n, k, experts, tiles_most, tile_rows, x_limit, steps, cblocks, n_cap, stages, tmem_cols, box, packed, lag, early, split, once;
    uint32_t *err;
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred q; elect.sync _|q, 0xffffffff; selp.u32 %0, 1, 0, q; }" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) { uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr)); return r; }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
template <int CG> __device__ __forceinline__ void i8_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    if constexpr (CG == 1) tma_load_2d(dst, map, bar, x, y);
    else asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int CG> __device__ __forceinline__ void i8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1) asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int CG> __device__ __forceinline__ void i8_commit(uint32_t bar) {   // in both CTAs of a pair
    if constexpr (CG == 1) tc_commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// 16 bytes to shared memory, zeros where `take` is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t take) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take) : "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
// 16 TMEM lanes x 16 columns: registers 4 i + {0, 1} hold lane T / 4, columns 8 i + 2 (T % 4) + {0, 1}; 4 i + {2, 3} the lane 8 further on
#define TMEM_LD16X256(taddr, r, o)                                                                                                       \
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"                                                 \
                 : "=r"(r[o + 0]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7]) : "r"(taddr))
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { uint32_t r; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}

// four sums and four of 64 channels further on at the same place of S CTAs' shared memory; all loads are on their way before the first is used
template <int S> __device__ __forceinline__ void i8_sum_parts(uint32_t addr, int (&sum)[8]) {
    int v[S][8];
#pragma unroll
    for (uint32_t r = 0; r < S; r++) {
        uint32_t from;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(addr), "r"(r));
        asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[r][0]), "=r"(v[r][1]), "=r"(v[r][2]), "=r"(v[r][3]) : "r"(from) : "memory");
        asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[r][4]), "=r"(v[r][5]), "=r"(v[r][6]), "=r"(v[r][7]) : "r"(from + 256u) : "memory");
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        sum[i] = 0;
#pragma unroll
        for (int r = 0; r < S; r++) sum[i] += v[r][i];
    }
}

struct I8Unit { uint32_t expert, row0, cnt, c0; };
// a place in a ring and the parity of its turn, without the divisions that a counter would need in every step (an issuer with them: 0.39 us per 128 columns, whatever the tile)
struct I8Stage { uint32_t s = 0, phase = 0; __device__ __forceinline__ void next(uint32_t count) { if (++s == count) { s = 0; phase ^= 1u; } } };
// Unit u is channel block u % cblocks of tile u / cblocks, and a worker takes every gridDim-th: the units in work at a time are those of neighbouring tiles, which share
// their rows and, where an expert has several tiles, its weights. (In runs of consecutive units per worker, cut by cost, an expert's weights came from memory once per tile: a
// 4096-token gate|up 159 us instead of 138.)
template <int CG> __device__ __forceinline__ I8Unit i8_unit(const I8MmaArgs &a, uint32_t u) {
    const uint32_t t = u / a.cblocks;
    I8Unit r;
    r.c0 = (u - t * a.cblocks) * (128u * CG);
    if (a.tiles) {   // of a plan that does not fit this call, what the call knows is bounded: experts, rows of a tile, rows of x and their scales. The lengths of maps and of y it does not know
        const uint4 v = a.tiles[t];
        r.expert = min(v.x, a.experts - 1u); r.row0 = v.y; r.cnt = min(min(v.z, a.tile_rows), a.x_limit > v.y ? a.x_limit - v.y : 0u);
    }
    else {   // 16 or 32 rows more or less, so that any number of tiles divides them evenly
        r.expert = 0; r.row0 = (uint32_t)((uint64_t)t * a.steps / a.tiles_most) * (16u * CG);
        r.cnt = min(a.m, (uint32_t)((uint64_t)(t + 1u) * a.steps / a.tiles_most) * (16u * CG)) - r.row0;
    }
    return r;
}

template <int CG, bool GATHER, bool SPLIT, int KPS>
__global__ void __launch_bounds__(i8_threads(GATHER), 1) i8_mma_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const I8MmaArgs a) {
    extern __shared__ uint8_t dyn_smem[];
    __shared__ __align__(8) uint64_t s_bar[2 * I8_STAGES + 5];
    __shared__ uint32_t s_tmem, s_abort, s_total;
    __shared__ __align__(16) float s_xs[2][I8_N_MAX];
    __shared__ __align__(16) uint32_t s_row[2][I8_N_MAX];
    __shared__ uint32_t s_src[GATHER ? 4 : 1][GATHER ? I8_N_MAX : 1];   // a copying warp's source rows of its unit
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, part = SPLIT || CG == 2 ? cluster_rank() : 0u, rank = CG == 2 ? part : 0u;   // part: of k, rank: of a pair
    const uint32_t smem_base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(s_bar);
    auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (I8_STAGES + s); };
    auto accfull_bar = [&](uint32_t b) { return bar0 + 8u * (2 * I8_STAGES + b); };
    auto accempty_bar = [&](uint32_t b) { return bar0 + 8u * (2 * I8_STAGES + 2 + b); };
    const uint32_t all_bar = bar0 + 8u * (2 * I8_STAGES + 4);   // every epilogue warp; not bar.sync, which would wait for a warp that gave up
    volatile uint32_t *abort_flag = &s_abort;
    const uint32_t x_tile = a.n_cap / CG * 128u, stage_bytes = KPS * (A_TILE + x_tile);   // KPS weight tiles, then KPS tiles of rows

    auto units = [&]() { return *reinterpret_cast<volatile uint32_t *>(a.err) ? 0u : (a.tiles ? min(a.header[2], a.tiles_most) : a.tiles_most) * a.cblocks; };   // after a recorded failure: no work

    if (threadIdx.x == 0) {
        s_abort = 0;
        if (a.early) s_total = units();
        // a filled stage: one arrival for the weights and one for the rows (of a pair by the first CTA, for both)
        for (uint32_t s = 0; s < I8_STAGES; s++) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }
        for (uint32_t b = 0; b < 2; b++) { mbar_init(accfull_bar(b), 1); mbar_init(accempty_bar(b), I8_EPI * CG); }
        mbar_init(all_bar, I8_EPI);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem, kb_all = (a.k + 128u * KPS - 1u) / (128u * KPS), kb0 = SPLIT ? kb_all * part / a.split : 0u, KB = SPLIT ? kb_all * (part + 1u) / a.split - kb0 : kb_all;   // this CTA's stages' columns
    if (!a.early || warp != 0) griddep_chain();   // early weights are requested while the kernels ahead still run
    const uint32_t total = a.early ? s_total : units();
    const uint32_t first = SPLIT ? blockIdx.x / a.split : blockIdx.x / CG, step = SPLIT ? gridDim.x : gridDim.x / CG;   // SPLIT: one unit
    auto tile_rows = [](uint32_t cnt) { return cnt ? (cnt + 16u * CG - 1u) / (16u * CG) * 16u : 16u; };   // rows of a tile that this CTA holds; a product has 16 at least, though a plan's tile may have none
    auto filled_bar = [&](uint32_t s) { return CG == 2 ? in_first_cta(full_bar(s)) : full_bar(s); };

    // Early weights' warp learns here that the kernels ahead are done, from warp 3, which has waited for them: a wait of its own so late takes 2 us (64 x 4096 x 4096: 7.7 -> 9.7)
    auto ahead_done = []() { asm volatile("barrier.sync 1, 64;" ::: "memory"); };
    if (a.early && warp == 3) asm volatile("barrier.arrive 1, 64;" ::: "memory");
    if (warp == 0) {
        // ---------------------------------------------------------------- weights
        const uint64_t policy = l2_policy_evict_first();
        I8Stage st; bool ok = true, waited = !a.early;
        for (uint32_t u = first; u < total && ok; u += step) {
            const I8Unit t = i8_unit<CG>(a, u);
            const int wy = (int)(t.expert * a.n + t.c0 + rank * 128u);
            for (uint32_t kb = 0; kb < KB; kb++, st.next(a.stages)) {
                if (!waited && st.phase) { ahead_done(); waited = true; }   // the ring is full: until the kernels ahead are done nothing empties it, and they may outlast a bounded wait
                if (!(ok = mbar_wait(empty_bar(st.s), st.phase ^ 1u, abort_flag, a.err, 1))) break;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full_bar(st.s), CG * KPS * A_TILE);
#pragma unroll
                    for (uint32_t h = 0; h < KPS; h++) {   // columns past the end are filled with zeros
                        const uint32_t dst = smem_base + st.s * stage_bytes + h * A_TILE; const int x = (int)(((kb0 + kb) * KPS + h) * 128u);
                        if (CG == 1 && a.once) tma_load_2d_hint(dst, &tm_w, full_bar(st.s), x, wy, policy); else i8_load<CG>(dst, &tm_w, filled_bar(st.s), x, wy);
                    }
                }
                __syncwarp();
            }
        }
        if (!waited) ahead_done();
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        // the whole warp walks through the loop, one lane issues: addresses and descriptors then stay in uniform registers
        I8Stage st, acc; bool ok = rank == 0;   // acc: accumulator buffers
        for (uint32_t u = first; u < total && ok; u += step, acc.next(2)) {
            const I8Unit t = i8_unit<CG>(a, u);
            const uint32_t cols = tile_rows(t.cnt) * CG, buf = acc.s;
            // D s32, A = B = signed 8-bit, both K-major, M 128 CG, N cols
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((cols >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
            const uint32_t d = tmem + buf * a.n_cap;
            if (!(ok = mbar_wait(accempty_bar(buf), acc.phase ^ 1u, abort_flag, a.err, 2))) break;
            tc_fence_after();
            for (uint32_t kb = 0; kb < KB; kb++, st.next(a.stages)) {
                if (!(ok = mbar_wait(full_bar(st.s), st.phase, abort_flag, a.err, 3))) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (uint32_t h = 0; h < KPS; h++) {
                        const uint64_t dw = umma_desc(smem_base + st.s * stage_bytes + h * A_TILE), dx = umma_desc(smem_base + st.s * stage_bytes + KPS * A_TILE + h * x_tile);
#pragma unroll
                        for (uint32_t ks = 0; ks < 4; ks++) i8_mma<CG>(d, dw + 2u * ks, dx + 2u * ks, idesc, kb | h | ks);   // 32 columns each
                    }
                    i8_commit<CG>(empty_bar(st.s));
                }
                __syncwarp();
            }
            if (ok && elect_one()) i8_commit<CG>(accfull_bar(buf));
            __syncwarp();
        }
    } else if (warp == 3) {
        // ---------------------------------------------------------------- activation rows
        if constexpr (!GATHER) {
            I8Stage st; bool ok = true;
            for (uint32_t u = first; u < total && ok; u += step) {
                const I8Unit t = i8_unit<CG>(a, u);
                const uint32_t rows = tile_rows(t.cnt), boxes = (rows + a.box - 1u) / a.box;
                const int y = (int)(t.row0 + rank * rows);
                for (uint32_t kb = 0; kb < KB; kb++, st.next(a.stages)) {
                    if (!(ok = mbar_wait(empty_bar(st.s), st.phase ^ 1u, abort_flag, a.err, 6))) break;
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx(full_bar(st.s), CG * KPS * boxes * a.box * 128u);
#pragma unroll
                        for (uint32_t h = 0; h < KPS; h++)
                            for (uint32_t i = 0; i < boxes; i++)
                                i8_load<CG>(smem_base + st.s * stage_bytes + KPS * A_TILE + h * x_tile + i * a.box * 128u, &tm_x, filled_bar(st.s), (int)(((kb0 + kb) * KPS + h) * 128u), y + (int)(i * a.box));
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= 4 && warp < 4 + I8_EPI) {
        // ---------------------------------------------------------------- epilogue: 32 channels and every fourth 16 rows per warp
        const uint32_t et = threadIdx.x - 128u, quarter = warp & 3u, sub = (warp - 4u) >> 2, out_base = smem_base + a.stages * stage_bytes + (warp - 4u) * I8_OUT;
        I8Unit next; float next_xs = 0.0f, next_w[4]; uint32_t next_row = 0;
        auto fetch = [&](uint32_t u) {   // what a unit's drain needs from memory, a unit ahead
            next = i8_unit<CG>(a, u);
            if (et < next.cnt) {
                const uint32_t r = next.row0 + et;
                next_xs = a.xs[a.xmap ? min(a.xmap[r], a.x_rows - 1u) : r];
                next_row = a.ymap ? a.ymap[r] : r;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t ch = next.c0 + rank * 128u + quarter * 32u + (a.packed ? (lane >> 2) + 8u * i : lane);
                next_w[i] = ch < a.n ? __ldg(a.ws + (size_t)next.expert * a.n + ch) : 0.0f;
            }
        };
        if (first < total) fetch(first);
        I8Stage acc; uint32_t n = 0; bool ok = true;
        for (uint32_t u = first; u < total && ok; u += step, n++, acc.next(2)) {
            const I8Unit t = next;
            const uint32_t buf = acc.s, p = n & 1u;
            if (et < t.cnt) { s_xs[p][et] = next_xs; s_row[p][et] = next_row; }
            float w[4];   // packed: channels lane / 4 + 0, 8, 16, 24 of the warp's 32; else [0]: channel lane
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = next_w[i];
            if (u + step < total) fetch(u + step);
            __syncwarp();
            if (lane == 0) mbar_arrive(all_bar);
            if (!(ok = mbar_wait(all_bar, n & 1u, abort_flag, a.err, 5))) break;
            if (!(ok = mbar_wait(accfull_bar(buf), acc.phase, abort_flag, a.err, 4))) break;
            tc_fence_after();
            // A pair's accumulator is handed back as soon as this warp's last load from it has landed (tcgen05.wait::ld), ahead of the results' way out. The arrival crosses to the other
            // CTA: it orders nothing but those loads, and releasing at cluster scope would wait for the stores before it to be acknowledged (a 4096-token layer's down product 78 us, 90
            // with a release after the stores). One CTA's is handed back after the stores have been issued: its units are many and short, and 64 tokens take 79 us so, 82 the other way.
            auto hand_back = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) { if constexpr (CG == 2) mbar_arrive_cluster_relaxed(in_first_cta(accempty_bar(buf))); else mbar_arrive(accempty_bar(buf)); }
            };
            if (CG == 2 && sub * 16u >= t.cnt) hand_back();   // no rows of this warp
            const uint32_t taddr = tmem + ((quarter * 32u) << 16) + buf * a.n_cap, ch0 = t.c0 + rank * 128u + quarter * 32u;
            if constexpr (SPLIT) {   // the stages have been read: their memory takes the sums, [row][channel]
                for (uint32_t c = sub * 16u; c < t.cnt; c += 64u) {
                    uint32_t v[16];
                    TMEM_LD16(taddr + c, v, 0);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (uint32_t i = 0; i < 16; i++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem_base + ((c + i) * 128u + quarter * 32u + lane) * 4u), "r"(v[i]) : "memory");
                }
            } else if (a.packed) {
                // a thread holds two neighbouring rows of a channel per register pair; the transposing store makes them 16-byte runs of a row's channels
                uint32_t v[16];
                const uint32_t part = lane & 3u, piece_ch = ch0 + part * 8u;
                if (sub * 16u < t.cnt) { TMEM_LD16X256(taddr + sub * 16u, v, 0); TMEM_LD16X256(taddr + (16u << 16) + sub * 16u, v, 8); }
                for (uint32_t c = sub * 16u; c < t.cnt; c += 64u) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (CG == 2 && c + 64u >= t.cnt) hand_back();
                    uint32_t o[8];
                    const float2 x0 = *reinterpret_cast<const float2 *>(&s_xs[p][c + 2u * part]), x1 = *reinterpret_cast<const float2 *>(&s_xs[p][c + 8u + 2u * part]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {   // 8 channels x 8 rows each: i & 1 the second eight channels, i >> 1 the second eight rows of the 16 x 16 block
                        const float2 x = i >> 1 ? x1 : x0;
                        o[i] = pack_bf16((float)(int)v[2 * i] * (x.x * w[i & 1]), (float)(int)v[2 * i + 1] * (x.y * w[i & 1]));
                        o[4 + i] = pack_bf16((float)(int)v[8 + 2 * i] * (x.x * w[2 + (i & 1)]), (float)(int)v[8 + 2 * i + 1] * (x.y * w[2 + (i & 1)]));
                    }
                    if (c + 64u < t.cnt) { TMEM_LD16X256(taddr + c + 64u, v, 0); TMEM_LD16X256(taddr + (16u << 16) + c + 64u, v, 8); }
                    const uint32_t at = out_base + ((lane >> 4) * 8u + (lane & 7u)) * I8_OUT_ROW + ((lane >> 3) & 1u) * 16u;
                    stmatrix_trans(at, o[0], o[1], o[2], o[3]);
                    stmatrix_trans(at + 32u, o[4], o[5], o[6], o[7]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t j = (lane >> 2) + 8u * i;
                        uint32_t q[4]; lds128(out_base + j * I8_OUT_ROW + part * 16u, q);
                        if (c + j < t.cnt && piece_ch < a.n) *reinterpret_cast<uint4 *>(a.y16 + (size_t)s_row[p][c + j] * a.n + piece_ch) = make_uint4(q[0], q[1], q[2], q[3]);
                    }
                    __syncwarp();
                }
            } else {
                for (uint32_t c = sub * 16u; c < t.cnt; c += 64u) {
                    uint32_t v[16];
                    TMEM_LD16(taddr + c, v, 0);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (CG == 2 && c + 64u >= t.cnt) hand_back();
                    if (ch0 + lane < a.n) {
#pragma unroll
                        for (uint32_t i = 0; i < 16; i++) {
                            if (c + i >= t.cnt) break;
                            const float y = (float)(int)v[i] * (s_xs[p][c + i] * w[0]);
                            const size_t at = (size_t)s_row[p][c + i] * a.n + ch0 + lane;
                            if (a.y16) a.y16[at] = (uint16_t)bf16_rne_bits(y);
                            if (a.y32) a.y32[at] = y;
                        }
                    }
                    __syncwarp();
                }
            }
            if (CG == 1) hand_back();
        }
    } else if (GATHER && warp >= 4 + I8_EPI) {
        // ---------------------------------------------------------------- row copies: each of the team's warps fills every team-th stage
        // No more warps than stages: a warp that waits for a place in the ring has then had one since the place's last turn began, and the barrier's parity tells the turns apart.
        constexpr uint32_t team = I8_TEAM;
        static_assert(I8_ROOM / (A_TILE + I8_N_MAX * 128) >= team, "a ring of as many stages as copying warps");
        // A stage is passed on once its copies have landed and are fenced for the tensor cores' reads; a.lag = 1: when the warp's next stage has been requested. In a ring of
        // 2 * team stages or more the place of stage i + team is free once stage i - team or an earlier one has been multiplied, which was passed on when stage i was requested.
        if constexpr (GATHER) {
            const uint32_t me = warp - (4 + I8_EPI), c = lane & 7u, r0 = lane >> 3;
            uint32_t *src = s_src[me];
            I8Stage st, done; bool ok = true, behind = false;
            uint32_t ahead[I8_N_MAX / 32] = {}, turn = 0;   // turn: stages until this warp's next
            for (uint32_t i = 0; i < me; i++) st.next(a.stages);
            done = st; turn = me;
            auto fetch = [&](uint32_t u) {
                const I8Unit t = i8_unit<CG>(a, u);
#pragma unroll
                for (uint32_t i = 0; i < I8_N_MAX / 32; i++) if (32u * i < t.cnt) ahead[i] = a.xmap[t.row0 + min(lane + 32u * i, t.cnt - 1u)];   // rows past the tile: any row, its columns are not read
                return tile_rows(t.cnt);
            };
            auto pass_on = [&]() {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(done.s));
                for (uint32_t i = 0; i < team; i++) done.next(a.stages);
            };
            uint32_t rows = first < total ? fetch(first) : 0u;
            for (uint32_t u = first; u < total && ok; u += step) {
                const uint32_t have = rows;
                __syncwarp();
#pragma unroll
                for (uint32_t i = 0; i < I8_N_MAX / 32; i++) if (32u * i < have) src[lane + 32u * i] = min(ahead[i], a.x_rows - 1u);
                __syncwarp();
                if (u + step < total) rows = fetch(u + step);   // a unit ahead: the map's values are there when they are needed
                for (uint32_t kb = turn; kb < KB; kb += team) {
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(st.s), st.phase ^ 1u, abort_flag, a.err, 7)))) break;
                    // the 128-byte swizzle: 16-byte column c of row r lies at column c ^ (r % 8)
#pragma unroll
                    for (uint32_t h = 0; h < KPS; h++) {
                        const uint32_t dst = smem_base + st.s * stage_bytes + KPS * A_TILE + h * x_tile, at = (kb * KPS + h) * 128u + c * 16u, take = at < a.k ? 16u : 0u;
                        const int8_t *from = a.x + (take ? at : 0u);
#pragma unroll 8
                        for (uint32_t r = r0; r < have; r += 4u) copy16(dst + r * 128u + ((c ^ (r & 7u)) << 4), from + (size_t)src[r] * a.x_stride, take);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (a.lag == 0u) { copies_wait<0>(); pass_on(); }
                    else if (behind) { copies_wait<1>(); pass_on(); }
                    else behind = true;
                    for (uint32_t i = 0; i < team; i++) st.next(a.stages);
                }
                turn = (turn + team - KB % team) % team;   // this warp's first stage of the next unit
            }
            copies_wait<0>();
            if (ok && behind) pass_on();
        }
    }
    if constexpr (SPLIT) {
        // ---------------------------------------------------------------- the parts' sums: every split-th row, two rows of 128 channels at a time per warp
        __syncwarp();
        cluster_sync();
        const uint32_t warps = blockDim.x / 32u, c = (lane & 15u) * 4u;
        if (first < total) {
            const I8Unit t = i8_unit<CG>(a, first);
            const uint32_t ch = t.c0 + c;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) { const uint32_t n = ch + (i & 3) + (i >> 2) * 64u; w[i] = n < a.n ? __ldg(a.ws + n) : 0.0f; }
            for (uint32_t j = part + a.split * (warp * 2u + (lane >> 4)); j < t.cnt; j += a.split * warps * 2u) {
                const float xs = a.xs[t.row0 + j];
                const uint32_t from = smem_base + (j * 128u + c) * 4u;
                int sum[8];
                if (a.split == 2u) i8_sum_parts<2>(from, sum); else if (a.split == 4u) i8_sum_parts<4>(from, sum); else i8_sum_parts<8>(from, sum);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t n = ch + h * 64u;
                    const size_t at = (size_t)(t.row0 + j) * a.n + n;
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = (float)sum[4 * h + i] * (xs * w[4 * h + i]);
                    if (a.packed) {
                        if (n < a.n) *reinterpret_cast<uint2 *>(a.y16 + at) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) if (n + i < a.n) { if (a.y16) a.y16[at + i] = (uint16_t)bf16_rne_bits(y[i]); if (a.y32) a.y32[at + i] = y[i]; }
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync();   // the other parts read this one's memory
    }
    // ---------------------------------------------------------------- teardown
    if (*abort_flag) { for (int i = 0; i < 64; i++) __nanosleep(1000); }   // let copies already issued land before the CTA goes away
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();   // the pair's products read this CTA's memory and arrive on its barriers
    if (warp == 2) {
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
    }
}

template <int CG, bool GATHER, bool SPLIT, int KPS>
static cudaError_t i8_mma_start(const CUtensorMap &w, const CUtensorMap &x, const I8MmaArgs &a, uint32_t grid, cudaStream_t s) {
    auto kernel = i8_mma_kernel<CG, GATHER, SPLIT, KPS>;
    // set on every call: it belongs to the device's context and costs well under a launch
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)I8_SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {}; cudaLaunchAttribute at[2];
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(i8_threads(GATHER)); cfg.dynamicSmemBytes = I8_SMEM; cfg.stream = s; cfg.attrs = at; cfg.numAttrs = SPLIT || CG == 2 ? 2 : 1;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension; at[1].val.clusterDim.x = SPLIT ? a.split : CG; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    return cudaLaunchKernelEx(&cfg, kernel, w, x, a);
}

// 128 or 256 columns in a stage. Two blocks halve the barriers' turns, which cost 0.04 us each; they want an even number of blocks in every part, and three stages, five where warps
// copy the rows (four of 64 rows: 66.1 us instead of 64.8). 300 x 4096 x 2048: 7.4 -> 6.7 us, 64 x 4096 x 4096: 7.8 -> 7.65, 64 tokens through 128 experts: gate|up 50.8 -> 50.0 and
// down 27.0 -> 26.0. Pairs take 0.25 us for a block's products alone: 4096 x 4096 x 4096 48.4 -> 49.3, so they stay with one.
static bool i8_two_blocks(uint32_t cg, uint32_t rows, uint32_t kb, uint32_t split, bool gather) {
    return cg == 1u && kb % (2u * (split > 1u ? split : 1u)) == 0u && I8_ROOM / (2u * (A_TILE + rows * 128u)) >= (gather ? 5u : 3u);
}

// Form and tile of a dense product: the least estimate, in us, over tile counts that divide the rows evenly. Measured with r rows in a tile, on L2-resident operands:
// 128 columns take 0.22 + 0.00042 r and at least 0.26 with one CTA (0.04 less where a stage holds two blocks), 0.15 + 0.0004 r and at least 0.19 with a pair, whose start costs 1.4 more; a unit's drain keeps a later one
// waiting from 0.5 + 0.013 r on and costs 0.2 + 0.008 r where none follows; a split costs 1.4 + 0.4 log2(parts) + 0.014 r. 64 x 4096 x 4096: 10.3 us in one part, 8.7 in two, 7.5 in
// four; 30 x 512 x 4096: 10.0, 8.1, 6.5, 5.8 in eight; 300 x 4096 x 2048: 7.6 with tiles of 80, 8.2 of 160, 11.0 of 64 (two rounds), 8.8 in pairs.
struct I8Form { uint32_t cg, tiles, split; };
static I8Form i8_dense_form(uint32_t m, uint32_t n, uint32_t k, uint32_t sms) {
    const uint32_t kb = (k + 127u) / 128u;
    I8Form f = {}; float best = 3.4e38f;
    for (uint32_t g = 1; g <= 2; g++) {
        const uint32_t blocks = (n + 128u * g - 1u) / (128u * g), steps = (m + 16u * g - 1u) / (16u * g), most = I8_N_MAX / (16u * g), least = (steps + most - 1u) / most, workers = sms / g;
        for (uint32_t t = least; t < least + 24u && t <= steps; t++) {
            const float r = (float)((steps + t - 1u) / t * (16u * g)), mean = fmaxf((float)m / t, 16.0f);   // rows of the longest tile, of all
            auto block = [&](uint32_t split) {
                return g == 1u ? fmaxf(0.26f, 0.22f + 0.00042f * mean) - (i8_two_blocks(g, (uint32_t)r, kb, split, false) ? 0.04f : 0.0f) : fmaxf(0.19f, 0.15f + 0.0004f * mean);
            };
            const float each = block(1u);
            const uint64_t units = (uint64_t)t * blocks;
            const float cost = (float)((units + workers - 1u) / workers) * fmaxf(kb * each, 0.5f + 0.013f * mean) + 0.2f + 0.008f * r + (g == 2u ? 1.4f : 0.0f);
            if (cost < best) { best = cost; f = {g, t, 1u}; }
            if (g == 2u) continue;
            uint32_t room = sms;   // clusters of 4 and 8 do not fill the SMs of every group that a cluster has to lie in: 16 of 8 took two rounds
            for (uint32_t s = 2, lg = 1; s <= 8u && s <= kb; s *= 2u, lg++, room -= sms / 8u) {
                if (units * s > room) break;
                const float split = (float)((kb + s - 1u) / s) * block(s) + 1.4f + 0.4f * lg + 0.014f * r;
                if (split < best) { best = split; f = {1u, t, s}; }
            }
        }
    }
    return f;
}

cudaError_t launch_i8_mma(const OmegaGpuI8Tensor *t, const I8Launch &l, cudaStream_t s) {
    const uint32_t sms = st().sm_count ? st().sm_count : 148;
    I8MmaArgs a = {};
    a.ws = t->s; a.xs = l.xs; a.y16 = l.y16; a.y32 = l.y32; a.tiles = (const uint4 *)l.tiles; a.header = l.header; a.xmap = l.xmap; a.ymap = l.ymap;
    a.m = l.m; a.n = l.n; a.k = t->k; a.experts = t->n / l.n; a.err = t->err; a.x = l.x; a.x_stride = l.x_stride ? l.x_stride : t->k; a.x_rows = l.x_rows; a.early = !l.tiles || l.early;
    // Tiles of few rows: hardly any expert has two. 64 tokens through 128 experts, gate|up 53 -> 50 us and down 29 -> 26 us; 4096 tokens in tiles of 256, 125 -> 134 and 78 -> 82.
    a.once = l.tiles && l.tile_rows <= 64u;
    uint32_t cg = 1;
    if (l.tiles) {
        a.tiles_most = l.m; a.tile_rows = l.tile_rows; a.x_limit = l.xmap ? 0xffffffffu : l.x_rows;
        cg = !l.xmap && l.tile_rows >= 128u ? 2u : 1u;   // long tiles in pairs: a layer of 4096 tokens 288 us instead of 307, of 1500 tokens 174 instead of 183
        a.n_cap = (l.tile_rows + 16u * cg - 1u) / (16u * cg) * (16u * cg);
    }
    else {
        const I8Form f = i8_dense_form(l.m, l.n, t->k, sms);
        cg = f.cg; a.split = f.split; a.tiles_most = f.tiles; a.steps = (l.m + 16u * cg - 1u) / (16u * cg);
        a.n_cap = (a.steps + f.tiles - 1u) / f.tiles * (16u * cg);
    }
    a.cblocks = (l.n + 128u * cg - 1u) / (128u * cg);
    const uint32_t per_cta = a.n_cap / cg;
    a.box = !l.tiles ? per_cta : per_cta % 64u == 0 ? 64u : per_cta % 32u == 0 ? 32u : 16u;
    a.packed = l.y16 && !l.y32 && l.n % 8u == 0;
    const bool two = i8_two_blocks(cg, per_cta, (t->k + 127u) / 128u, a.split, l.xmap != nullptr);
    a.stages = I8_ROOM / ((A_TILE + per_cta * 128u) * (two ? 2u : 1u)); if (a.stages > I8_STAGES) a.stages = I8_STAGES;
    a.lag = a.stages >= 2u * I8_TEAM;
    a.tmem_cols = 32; while (a.tmem_cols < 2u * a.n_cap) a.tmem_cols *= 2;
    CUtensorMap w, x;
    if (!make_tmap_u8(&w, t->w, t->n, t->k, 128) || !make_tmap_u8(&x, l.x, l.x_rows, t->k, a.box, l.x_stride)) return cudaErrorInvalidValue;
    const uint64_t units = (uint64_t)a.tiles_most * a.cblocks;
    if (units > 0x7fffffffull) return cudaErrorInvalidValue;
    uint32_t grid = a.split > 1u ? (uint32_t)units * a.split : (uint32_t)(units * cg < sms ? units * cg : sms); grid -= grid % cg;
    if (cg == 2u) return i8_mma_start<2, false, false, 1>(w, x, a, grid, s);
#define I8_START(GATHER, SPLIT) return two ? i8_mma_start<1, GATHER, SPLIT, 2>(w, x, a, grid, s) : i8_mma_start<1, GATHER, SPLIT, 1>(w, x, a, grid, s)
    if (a.split > 1u) I8_START(false, true);
    if (l.xmap) I8_START(true, false);
    I8_START(false, false);
#undef I8_START
}

}  // namespace b200
