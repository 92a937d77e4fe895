// moe_score_route.cu: routing by scores: softmax or sigmoid scores, a bias that only the selection sees, groups of experts of which the best are kept, top-k,
// weights renormalised over the picks.
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  c_e = s_e + b_e;  rank of a group = sum of its one or two largest c;  picks = topk largest c of the kept groups;
//   w = s / (sum of the picks' s + 1e-20) * weight_scale.
//
// Scores are computed in binary64 and rounded once to f32. Two experts whose c differ by an ulp would else change places with the exponential of the day (about
// one token in 5000 at 256 experts), and the ids are exact values that a caller compares. The picks are then made on 32-bit keys in the floats' order, which
// one redux instruction per round reduces.
#include <math.h>
#include "internal.h"

namespace b200 {

struct RouteArgs {
    const void *logits; const float *bias; uint32_t *ids; float *wts;
    size_t stride;                       // bytes between rows of logits
    uint32_t tokens, experts, topk, groups, kept, rank2, size;   // size = experts / groups
    int bf16, sigmoid, norm, vec;
    float scale;
};

constexpr uint32_t ROUTE_WARPS = 4;
constexpr uint32_t KEY_NAN = 1;          // below the key of -infinity; 0 = not to be picked
__device__ __forceinline__ uint32_t order_key(float v) {   // larger float, larger key; NaN lowest
    if (v != v) return KEY_NAN;
    const uint32_t b = __float_as_uint(v + 0.0f);          // -0 becomes +0: they are equal
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ void push_top2(float v, float &a, float &b) { if (v > a) { b = a; a = v; } else if (v > b) b = v; }

// One warp per token; a lane holds the VPL consecutive experts from lane * VPL, so the lowest lane of equal keys holds the lowest index.
template <int VPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) score_route_kernel(const RouteArgs a) {
    griddep_chain();
    extern __shared__ float route_sm[];   // [warp][experts], only where groups do not fall on whole lanes
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
    float s[VPL];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = l[i] != l[i] ? 0.0f : (float)(1.0 / (1.0 + exp(-(double)l[i])));
    } else {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < VPL; i++) top = fmaxf(top, l[i]);   // drops NaN
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        double e[VPL], sum = 0.0;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            e[i] = l[i] != l[i] || l[i] == -INFINITY ? 0.0 : l[i] == top ? 1.0 : exp((double)l[i] - (double)top);   // l == top also where both are +infinity
            sum += e[i];
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = sum > 0.0 ? (float)(e[i] / sum) : 0.0f;
    }
    uint32_t key[VPL];
    float c[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const uint32_t e = e0 + i;
        c[i] = a.bias && e < a.experts ? s[i] + a.bias[e] : s[i];
        if (l[i] != l[i]) c[i] = NAN;
        key[i] = e < a.experts ? order_key(c[i]) : 0u;
    }
    if (a.kept < a.groups) {
        // rank of group g on lane g
        float rank = -INFINITY;
        const uint32_t span = a.size / VPL;   // lanes of a group, where it falls on whole lanes
        if (a.size % VPL == 0 && (span & (span - 1u)) == 0u) {
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
            float *cs = route_sm + warp * a.experts;
#pragma unroll
            for (int i = 0; i < VPL; i++) if (e0 + i < a.experts) cs[e0 + i] = c[i];
            __syncwarp();
            if (lane < a.groups) {
                float x = -INFINITY, y = -INFINITY;
                for (uint32_t i = 0; i < a.size; i++) push_top2(cs[lane * a.size + i], x, y);
                rank = a.rank2 ? x + y : x;
            }
        }
        uint32_t gkey = lane < a.groups ? order_key(rank) : 0u, keep = 0;
        for (uint32_t r = 0; r < a.kept; r++) {
            const uint32_t best = __reduce_max_sync(0xffffffffu, gkey);
            const uint32_t who = __ffs(__ballot_sync(0xffffffffu, gkey == best)) - 1;
            keep |= 1u << who;
            if (lane == who) gkey = 0;
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) if (e0 + i < a.experts && !((keep >> ((e0 + i) / a.size)) & 1u)) key[i] = 0;
    }
    uint32_t my_id = 0; float my_s = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPL; i++) top = max(top, key[i]);
    for (uint32_t r = 0; r < a.topk; r++) {
        const uint32_t best = __reduce_max_sync(0xffffffffu, top);
        const uint32_t who = __ffs(__ballot_sync(0xffffffffu, top == best)) - 1;
        uint32_t at = 0; float sv = 0.0f;
#pragma unroll
        for (int i = VPL - 1; i >= 0; i--) if (key[i] == best) { at = i; sv = s[i]; }
        if (lane == who) {
            top = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) { if ((uint32_t)i == at) key[i] = 0; top = max(top, key[i]); }
        }
        const uint32_t id = __shfl_sync(0xffffffffu, e0 + at, who);
        sv = __shfl_sync(0xffffffffu, sv, who);
        if (lane == r) { my_id = id; my_s = sv; }
    }
    float sum = lane < a.topk ? my_s : 0.0f;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < a.topk) {
        a.ids[(size_t)t * a.topk + lane] = my_id;
        a.wts[(size_t)t * a.topk + lane] = (a.norm ? __fdiv_rn(my_s, sum + 1e-20f) : my_s) * a.scale;
    }
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

cudaError_t launch_score_route(const OmegaGpuMoeRouteConfig &c, uint32_t tokens, const void *logits, int bf16, size_t stride, const float *bias, uint32_t *ids, float *wts, cudaStream_t s) {
    RouteArgs a = {};
    const uint32_t elem = bf16 ? 2u : 4u;
    a.logits = logits; a.bias = bias; a.ids = ids; a.wts = wts; a.stride = stride ? stride : (size_t)c.experts * elem;
    a.tokens = tokens; a.experts = c.experts; a.topk = c.topk; a.groups = c.groups ? c.groups : 1u; a.kept = c.topk_groups ? c.topk_groups : a.groups;
    a.rank2 = c.group_rank == 2u; a.size = c.experts / a.groups;
    a.bf16 = bf16; a.sigmoid = c.score == OMEGA_GPU_MOE_SCORE_SIGMOID; a.norm = c.norm_topk != 0; a.scale = c.weight_scale;
    const uint32_t vpl = c.experts <= 128 ? 4u : c.experts <= 256 ? 8u : c.experts <= 512 ? 16u : 32u;
    a.vec = ((uintptr_t)logits % 16u) == 0 && a.stride % 16u == 0 && c.experts % vpl == 0;
    const size_t smem = a.kept < a.groups ? (size_t)ROUTE_WARPS * c.experts * 4 : 0;
    const dim3 grid((tokens + ROUTE_WARPS - 1) / ROUTE_WARPS), block(ROUTE_WARPS * 32);
    return vpl == 4u ? launch_chained(score_route_kernel<4>, grid, block, smem, s, a) : vpl == 8u ? launch_chained(score_route_kernel<8>, grid, block, smem, s, a)
         : vpl == 16u ? launch_chained(score_route_kernel<16>, grid, block, smem, s, a) : launch_chained(score_route_kernel<32>, grid, block, smem, s, a);
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
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return cuda_ok(launch_score_route(*cfg, tokens, (const void *)(uintptr_t)logits_va, logits_bf16 != 0, logits_stride_bytes, (const float *)(uintptr_t)bias_va, (uint32_t *)(uintptr_t)ids_va,
                                      (float *)(uintptr_t)wts_va, (cudaStream_t)stream), "route launch") ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_moe_route(const OmegaGpuMoeRouteConfig *cfg, uint32_t tokens, const void *logits, int logits_bf16, const float *bias, uint32_t *ids, float *wts) {
    const int rc = route_check(cfg);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    if (!tokens || !logits || !ids || !wts) return OMEGA_GPU_FP8_BAD_ARGS;
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
