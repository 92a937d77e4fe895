// moe_score_route.cu: routing by scores: softmax or sigmoid scores, a bias that only the selection sees, groups of experts of which the best are kept, top-k,
// weights renormalised over the picks.
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  c_e = s_e + b_e;  rank of a group = sum of its one or two largest c;  picks = topk largest c of the kept groups;
//   w = s / (sum of the picks' s + 1e-20) * weight_scale.
//
// The picks are those of scores computed in binary64 and rounded once to f32: two experts whose c differ by an ulp would else change places with the exponential of the day
// (about one token in 5000 at 256 experts), and the ids are exact values that a caller compares. A first pass takes f32 scores and looks for the few experts that can
// be among the picks, by more than the scores' error bound; those, one per lane, get their scores in binary64 and are ranked. Where the f32 scores do not decide which
// groups are kept, or more than 32 experts are as good as equal, a second pass does it all in binary64. Values are ordered as 32-bit keys, which one redux instruction
// reduces. 8192 tokens x 256 experts in groups: 14.2 us, bound by instruction issue (about 1100 a token; the 9 MB of memory traffic would take 1.5 us); 17.7 with
// binary64 scores for every expert. One token: 4.0 us.
#include <math.h>
#include "internal.h"

namespace b200 {

struct RouteArgs {
    const void *logits; const float *bias; uint32_t *ids; float *wts;
    size_t stride;                       // bytes between rows of logits
    uint32_t tokens, experts, topk, groups, kept, rank2, size;   // size = experts / groups
    int bf16, sigmoid, norm, vec, bias_vec;
    uint4 *tiles; uint32_t *header, *xmap, *ymap;   // one token: its routing plan as well, or null
    uint32_t magic;                      // e / size = umulhi(e, magic) for e < 1024, size > 1
    float scale;
};

constexpr uint32_t ROUTE_WARPS = 4, ROUTE_MOST_TOKENS = 1u << 30;
constexpr float TINY = 1e-36f;           // below it f32 scores may have lost their relative error bound: subnormal numbers, and quotients of 2^126 and more
constexpr uint32_t KEY_NAN = 1;          // below the key of -infinity; 0 = not to be picked
__device__ __forceinline__ uint32_t order_key(float v) {   // larger float, larger key; NaN lowest
    const uint32_t b = __float_as_uint(v);                 // never -0: scores are not, and a sum is only where both parts are
    return v != v ? KEY_NAN : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ void push_top2(float v, float &a, float &b) { if (v > a) { b = a; a = v; } else if (v > b) b = v; }

// One warp per token; a lane holds the VPL consecutive experts from lane * VPL, so the lowest lane of equal keys holds the lowest index. FINE: softmax weights that are not
// renormalised carry the error of the sum, so its exponentials are better ones (8192 tokens x 256 experts 17.3 us; 16.0 with the fast ones, which the others keep).
template <int VPL, bool FINE>
__global__ void __launch_bounds__(ROUTE_WARPS * 32, VPL <= 8 ? 8 : 2) score_route_kernel(const RouteArgs a) {
    griddep_chain();
    extern __shared__ float route_sm[];   // [warp][experts]
    __shared__ uint64_t s_cand[ROUTE_WARPS][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = blockIdx.x * ROUTE_WARPS + warp;
    if (t >= a.tokens) return;
    const uint32_t e0 = lane * VPL;
    float l[VPL];
    const uint8_t *row = static_cast<const uint8_t *>(a.logits) + (size_t)t * a.stride;
    if (a.vec) {   // rows on 16 bytes and experts % VPL == 0: a lane's block is wholly inside or outside
#pragma unroll
        for (int i = 0; i < VPL; i++) l[i] = -INFINITY;
        if (e0 < a.experts) {
            if (a.bf16) {
#pragma unroll
                for (int i = 0; i < VPL; i += 4) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(row + (e0 + i) * 2u);
                    l[i] = __uint_as_float(w.x << 16); l[i + 1] = __uint_as_float(w.x & 0xffff0000u); l[i + 2] = __uint_as_float(w.y << 16); l[i + 3] = __uint_as_float(w.y & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VPL; i += 4) { const float4 w = *reinterpret_cast<const float4 *>(row + (e0 + i) * 4u); l[i] = w.x; l[i + 1] = w.y; l[i + 2] = w.z; l[i + 3] = w.w; }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const uint32_t e = e0 + i;
            l[i] = e >= a.experts ? -INFINITY : a.bf16 ? __uint_as_float((uint32_t) reinterpret_cast<const uint16_t *>(row)[e] << 16) : reinterpret_cast<const float *>(row)[e];
        }
    }
    float top = -INFINITY;
    if (!a.sigmoid) {
#pragma unroll
        for (int i = 0; i < VPL; i++) top = fmaxf(top, l[i]);   // drops NaN
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const int inside = e0 >= a.experts ? 0 : a.experts - e0 < VPL ? (int)(a.experts - e0) : VPL;   // experts of this lane
    float bias[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) bias[i] = 0.0f;
    if (a.bias_vec) {
        if (e0 < a.experts) {
#pragma unroll
            for (int i = 0; i < VPL; i += 4) { const float4 b = *reinterpret_cast<const float4 *>(a.bias + e0 + i); bias[i] = b.x; bias[i + 1] = b.y; bias[i + 2] = b.z; bias[i + 3] = b.w; }
        }
    } else if (a.bias) {
#pragma unroll
        for (int i = 0; i < VPL; i++) if (e0 + i < a.experts) bias[i] = a.bias[e0 + i];
    }
    float s[VPL];
    double sum = 0.0;      // of the softmax
    uint32_t my_id = 0, my_rank = lane; float my_s = 0.0f;   // a pick and its place
    float *cs = route_sm + warp * a.experts + e0;   // this lane's values
    // a score's part in binary64; l == top also where both are +infinity
    auto score = [&](float v) {
        if (v != v) return 0.0;
        if (a.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
        return v == -INFINITY ? 0.0 : v == top ? 1.0 : exp((double)v - (double)top);
    };
    // e^(v - top), off by 3e-7 at most: 2 units of 2^-23 of expf and half a unit of the product with what the subtraction lost
    auto below_top = [&](float v) {
        const float d = v - top, t = d - v, lost = (v - (d - t)) - (top + t), e = expf(d);   // d + lost = v - top exactly, where d is finite
        return e > 0.0f ? fmaf(e, lost, e) : 0.0f;
    };
#pragma unroll 1
    for (int exact = 0; exact < 2; exact++) {
        sum = 0.0;
        if (exact) {   // two values at a time through shared memory: unrolled, this rare pass would take the registers of the common one
#pragma unroll
            for (int i = 0; i < VPL; i++) if (e0 + i < a.experts) cs[i] = l[i];
            double all = 1.0;
            if (!a.sigmoid) {
#pragma unroll 2
                for (uint32_t i = 0; i < VPL && e0 + i < a.experts; i++) sum += score(cs[i]);
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                all = sum > 0.0 ? sum : 1.0;
            }
#pragma unroll 2
            for (uint32_t i = 0; i < VPL && e0 + i < a.experts; i++) cs[i] = a.sigmoid ? (float)score(cs[i]) : (float)(score(cs[i]) / all);
#pragma unroll
            for (int i = 0; i < VPL; i++) s[i] = e0 + i < a.experts ? cs[i] : 0.0f;
        } else if (a.sigmoid) {
#pragma unroll
            for (int i = 0; i < VPL; i++) s[i] = __fdividef(1.0f, 1.0f + __expf(-l[i]));   // NaN stays NaN
        } else {
#pragma unroll
            for (int i = 0; i < VPL; i++) { s[i] = l[i] != l[i] || l[i] == -INFINITY ? 0.0f : l[i] == top ? 1.0f : FINE ? below_top(l[i]) : __expf(l[i] - top); sum += (double)s[i]; }
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = sum > 0.0 ? (float)(1.0 / sum) : 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; i++) s[i] *= inv;
        }
        uint32_t key[VPL];
        float c[VPL];
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            c[i] = a.sigmoid && !exact ? s[i] + bias[i] : l[i] != l[i] ? NAN : s[i] + bias[i];
            key[i] = i < inside ? order_key(c[i]) : 0u;
        }
        const float most = a.sigmoid ? 1.0f : sum > 0.0 ? (float)(1.0 / sum) : 1.0f;   // no score is larger
        bool near = false;   // f32 scores do not decide
        if (a.kept < a.groups) {
            // rank of group g on lane g
            float rank = -INFINITY;
            const uint32_t span = a.size / VPL;   // lanes of a group, where it falls on whole lanes
            const bool whole = a.size % VPL == 0 && (span & (span - 1u)) == 0u;
            if (whole) {
                float x = -INFINITY, y = -INFINITY;
#pragma unroll
                for (int i = 0; i < VPL; i++) push_top2(c[i], x, y);   // comparisons with NaN are false: it counts as the lowest
                for (uint32_t o = 1; o < span; o <<= 1) {
                    const float ox = __shfl_xor_sync(0xffffffffu, x, o), oy = __shfl_xor_sync(0xffffffffu, y, o);
                    push_top2(ox, x, y); push_top2(oy, x, y);
                }
                const float r = a.rank2 ? x + y : x;
                rank = __shfl_sync(0xffffffffu, r, (lane * span) & 31u);
            } else {
                const float *all = route_sm + warp * a.experts;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < VPL; i++) if (e0 + i < a.experts) cs[i] = c[i];
                __syncwarp();
                if (lane < a.groups) {
                    float x = -INFINITY, y = -INFINITY;
                    for (uint32_t i = 0; i < a.size; i++) push_top2(all[lane * a.size + i], x, y);
                    rank = a.rank2 ? x + y : x;
                }
                __syncwarp();
            }
            uint32_t gkey = lane < a.groups ? order_key(rank) : 0u, keep = 0, who = 0;
            for (uint32_t r = 0; r < a.kept; r++) {
                const uint32_t best = __reduce_max_sync(0xffffffffu, gkey);
                who = __ffs(__ballot_sync(0xffffffffu, gkey == best)) - 1;
                keep |= 1u << who;
                if (lane == who) gkey = 0;
            }
            const uint32_t next = __reduce_max_sync(0xffffffffu, gkey);
            const float in = __shfl_sync(0xffffffffu, rank, who), out = __shfl_sync(0xffffffffu, rank, __ffs(__ballot_sync(0xffffffffu, gkey == next)) - 1);
            near = !(in - out > 5e-6f * most + 5e-7f * (fabsf(in) + fabsf(out)));   // four f32 scores and the roundings of their sums
            if (whole) {
                if (!((keep >> (lane >> (31 - __clz(span)))) & 1u)) {
#pragma unroll
                    for (int i = 0; i < VPL; i++) key[i] = 0;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VPL; i++) if (!((keep >> (a.size > 1u ? __umulhi(e0 + i, a.magic) : e0 + i)) & 1u)) key[i] = 0;   // past the experts it is 0 anyway
            }
        }
        if (!exact) {
            // Candidates: what is not below the topk-th largest of the lanes' best, which is no more than the topk-th largest of all, by more than two scores' error. Of f32 scores
            // the exponential of x is off by (2 + 1.173 |x|) 2^-23, quotient and sums by 2 units: less than 2e-5 of a score that is no subnormal, and, as
            // |x| e^-|x| < 0.4, less than 7e-7 of the largest score.
            uint32_t m = 0, least = 1;
#pragma unroll
            for (int i = 0; i < VPL; i++) m = max(m, key[i]);
            for (uint32_t r = 0; r < a.topk; r++) {
                const uint32_t best = __reduce_max_sync(0xffffffffu, m);
                least = max(best, 1u);   // fewer lanes with experts than that: all of theirs
                if (m == best) m = 0;
            }
            const float edge = key_value(least);
            if (least > KEY_NAN && fabsf(edge) <= 3.0e38f) least = order_key(a.bias ? edge - (4e-6f * most + 5e-7f * fabsf(edge)) : edge < TINY ? 0.0f : edge - 1e-4f * edge);
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const uint32_t those = __ballot_sync(0xffffffffu, key[i] >= least), at = n + __popc(those & ((1u << lane) - 1u));
                if (key[i] >= least && at < 32u) s_cand[warp][at] = e0 + i;
                n += __popc(those);
            }
            __syncwarp();
            if (n <= 32u) {
                uint64_t mine = 0;
                float my_l = -INFINITY;
                if (lane < n) {
                    const uint32_t e = (uint32_t)s_cand[warp][lane];
                    const float v = a.bf16 ? __uint_as_float((uint32_t) reinterpret_cast<const uint16_t *>(row)[e] << 16) : reinterpret_cast<const float *>(row)[e];
                    my_id = e; my_l = v;
                    my_s = a.sigmoid ? (float)score(v) : (float)(score(v) / (sum > 0.0 ? sum : 1.0));
                    mine = ((uint64_t)order_key(v != v ? v : a.bias ? my_s + a.bias[e] : my_s) << 32) | ~e;   // ~e: the lowest index of equals first
                }
                __syncwarp();
                if (lane < n) s_cand[warp][lane] = mine;
                __syncwarp();
                uint32_t place = 0;
                for (uint32_t j = 0; j < n; j++) place += s_cand[warp][j] > mine;
                my_rank = lane < n ? place : 32u;
                if (!a.sigmoid) {
                    // The softmax's sum may be of f32 exponentials, off by (2 + 1.173 |x|) 2^-23 each and by |x| 2^-24 with the subtraction's rounding: where 1023 experts share one logit, |x| = 5.4
                    // makes the most of it, 1.1e-6 of the sum. Neighbours that this could make equal, or no longer equal, are left to the second pass; without a bias the sum's error is a
                    // factor of both and only their roundings count
                    __syncwarp();
                    if (lane < n) s_cand[warp][place] = mine;
                    __syncwarp();
                    // (rounded to a subnormal number, that much of a score may be a whole unit of it)
                    if (!a.bias && lane < n && place < a.topk && (uint32_t)(mine >> 32) > KEY_NAN) near |= my_s < TINY && my_l != -INFINITY;
                    const uint64_t next = place < a.topk && place + 1u < n ? s_cand[warp][place + 1u] : 0;
                    if ((uint32_t)(next >> 32) > KEY_NAN) {
                        const float v = key_value((uint32_t)(mine >> 32)), w = key_value((uint32_t)(next >> 32));
                        near |= v != w && !(v - w > (a.bias ? 1.5e-6f * most : 1e-6f * my_s) + (a.bias ? 2.4e-7f * fabsf(v) : 0.0f));
                        // equal as they are: the same logit and bias, or near
                        if (v == w) {
                            const uint32_t e = my_id, f = ~(uint32_t)next;
                            const bool same_l = a.bf16 ? reinterpret_cast<const uint16_t *>(row)[e] == reinterpret_cast<const uint16_t *>(row)[f] : reinterpret_cast<const float *>(row)[e] == reinterpret_cast<const float *>(row)[f];
                            near |= !(same_l && (!a.bias || a.bias[e] == a.bias[f]));
                        }
                    }
                }
                if (!__any_sync(0xffffffffu, near)) break;
                my_rank = lane;
            }
            __syncwarp();
            continue;
        }
        // each lane's best: key, place, value; the winner of a round looks for its next
        uint32_t best_key = 0, best_i = 0;
        auto look = [&]() {
            best_key = 0; best_i = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) if (key[i] > best_key) { best_key = key[i]; best_i = i; }
        };
        look();
        for (uint32_t r = 0; r < a.topk; r++) {
            const uint32_t best = __reduce_max_sync(0xffffffffu, best_key);
            const uint32_t who = __ffs(__ballot_sync(0xffffffffu, best_key == best)) - 1;
            float ws = 0.0f;
            uint32_t id = 0;
            if (lane == who) {
#pragma unroll
                for (int i = 0; i < VPL; i++) if ((uint32_t)i == best_i) { ws = s[i]; key[i] = 0; }
                id = e0 + best_i;
                look();
            }
            id = __shfl_sync(0xffffffffu, id, who); ws = __shfl_sync(0xffffffffu, ws, who);
            if (lane == r) { my_id = id; my_s = ws; }
        }
    }
    const bool pick = my_rank < a.topk;
    float total = pick ? my_s : 0.0f;
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (pick) {
        a.ids[(size_t)t * a.topk + my_rank] = my_id;
        a.wts[(size_t)t * a.topk + my_rank] = (a.norm ? __fdiv_rn(my_s, total + 1e-20f) : my_s) * a.scale;
        if (a.tiles) {   // every pick is a tile of one row, in the picks' order
            a.tiles[my_rank] = make_uint4(my_id, my_rank, 1u, my_rank);
            a.xmap[my_rank] = 0; a.ymap[my_rank] = my_rank;
            if (my_rank < 4u) a.header[my_rank] = my_rank < 3u ? a.topk : 0u;
        }
    }
    if (a.tiles && lane < 4u && a.topk <= lane) a.header[lane] = lane < 3u ? a.topk : 0u;   // fewer than four picks
}

static int route_check(const OmegaGpuMoeRouteConfig *c) {
    if (!c || !c->experts || c->experts > 1024 || !c->topk || c->topk > 32 || c->score > OMEGA_GPU_MOE_SCORE_SIGMOID || c->group_rank > 2) return OMEGA_GPU_FP8_BAD_ARGS;
    const uint32_t groups = c->groups ? c->groups : 1u, kept = c->topk_groups ? c->topk_groups : groups, rank = c->group_rank ? c->group_rank : 1u;
    if (groups > 32 || c->experts % groups || kept > groups) { set_error("route: %u groups (%u kept) of %u experts", groups, kept, c->experts); return OMEGA_GPU_FP8_BAD_ARGS; }
    const uint32_t size = c->experts / groups;
    if (rank > size || c->topk > kept * size) { set_error("route: %u picks and a rank of %u from %u groups of %u experts", c->topk, rank, kept, size); return OMEGA_GPU_FP8_BAD_ARGS; }
    if (!(fabsf(c->weight_scale) <= 3.0e38f)) { set_error("route: weight_scale is not finite"); return OMEGA_GPU_FP8_BAD_ARGS; }
    return OMEGA_GPU_FP8_OK;
}
int score_route_ok(const OmegaGpuMoeRouteConfig *c) { return route_check(c); }

cudaError_t launch_score_route(const OmegaGpuMoeRouteConfig &c, uint32_t tokens, const void *logits, int bf16, size_t stride, const float *bias, uint32_t *ids, float *wts, cudaStream_t s,
                               const OmegaGpuMoePlanOut *plan) {
    RouteArgs a = {};
    if (plan && tokens == 1u) { a.tiles = (uint4 *)(uintptr_t)plan->tiles_va; a.header = (uint32_t *)(uintptr_t)plan->header_va; a.xmap = (uint32_t *)(uintptr_t)plan->xmap_va; a.ymap = (uint32_t *)(uintptr_t)plan->ymap_va; }
    const uint32_t elem = bf16 ? 2u : 4u;
    a.logits = logits; a.bias = bias; a.ids = ids; a.wts = wts; a.stride = stride ? stride : (size_t)c.experts * elem;
    a.tokens = tokens; a.experts = c.experts; a.topk = c.topk; a.groups = c.groups ? c.groups : 1u; a.kept = c.topk_groups ? c.topk_groups : a.groups;
    a.rank2 = c.group_rank == 2u; a.size = c.experts / a.groups;
    a.bf16 = bf16; a.sigmoid = c.score == OMEGA_GPU_MOE_SCORE_SIGMOID; a.norm = c.norm_topk != 0; a.scale = c.weight_scale;
    const uint32_t vpl = c.experts <= 128 ? 4u : c.experts <= 256 ? 8u : c.experts <= 512 ? 16u : 32u;
    a.vec = ((uintptr_t)logits % 16u) == 0 && a.stride % 16u == 0 && c.experts % vpl == 0;
    a.bias_vec = bias && ((uintptr_t)bias % 16u) == 0 && c.experts % vpl == 0; a.magic = a.size > 1u ? 0xffffffffu / a.size + 1u : 0u;
    const size_t smem = (size_t)ROUTE_WARPS * c.experts * 4;
    const dim3 grid((tokens + ROUTE_WARPS - 1) / ROUTE_WARPS), block(ROUTE_WARPS * 32);
#define ROUTE(VPL) return !a.sigmoid && !a.norm ? launch_chained(score_route_kernel<VPL, true>, grid, block, smem, s, a) : launch_chained(score_route_kernel<VPL, false>, grid, block, smem, s, a)
    if (vpl == 4u) ROUTE(4);
    if (vpl == 8u) ROUTE(8);
    if (vpl == 16u) ROUTE(16);
    ROUTE(32);
#undef ROUTE
}

}  // namespace b200
using namespace b200;

extern "C" {

int omega_gpu_moe_route_async(const OmegaGpuMoeRouteConfig *cfg, uint32_t tokens, uint64_t logits_va, int logits_bf16, uint32_t logits_stride_bytes, uint64_t bias_va,
                              uint64_t ids_va, uint64_t wts_va, void *stream) {
    const int rc = route_check(cfg);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    const uint32_t elem = logits_bf16 ? 2u : 4u;
    if (!tokens || !logits_va || !ids_va || !wts_va || ((ids_va | wts_va | bias_va) & 3u) || logits_va % elem) return OMEGA_GPU_FP8_BAD_ARGS;
    if (logits_stride_bytes && (logits_stride_bytes % elem || logits_stride_bytes < cfg->experts * elem)) { set_error("route: rows of logits %u bytes apart", logits_stride_bytes); return OMEGA_GPU_FP8_BAD_ARGS; }
    if (tokens > ROUTE_MOST_TOKENS) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return cuda_ok(launch_score_route(*cfg, tokens, (const void *)(uintptr_t)logits_va, logits_bf16 != 0, logits_stride_bytes, (const float *)(uintptr_t)bias_va, (uint32_t *)(uintptr_t)ids_va,
                                      (float *)(uintptr_t)wts_va, (cudaStream_t)stream), "route launch") ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_moe_route(const OmegaGpuMoeRouteConfig *cfg, uint32_t tokens, const void *logits, int logits_bf16, const float *bias, uint32_t *ids, float *wts) {
    const int rc = route_check(cfg);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    if (!tokens || !logits || !ids || !wts) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > ROUTE_MOST_TOKENS) return OMEGA_GPU_FP8_TOO_LARGE;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    const size_t lb = (size_t)tokens * cfg->experts * (logits_bf16 ? 2 : 4), ib = (size_t)tokens * cfg->topk * 4, bb = (size_t)cfg->experts * 4;
    void *dl = stage(0, lb); uint32_t *di = (uint32_t *)stage(1, ib); float *dw = (float *)stage(2, ib), *db = (float *)stage(3, bb);
    if (!dl || !di || !dw || !db) return OMEGA_GPU_FP8_CHIP_FAIL;
    cudaStream_t s = st().stream;
    const bool ok = to_device(dl, logits, lb, s) && (!bias || to_device(db, bias, bb, s)) &&
                    cuda_ok(launch_score_route(*cfg, tokens, dl, logits_bf16 != 0, 0, bias ? db : nullptr, di, dw, s), "route launch") && to_host(ids, di, ib, s) && to_host(wts, dw, ib, s) &&
                    cuda_ok(cudaStreamSynchronize(s), "route");
    return ok ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

}  // extern "C"
