// moe_i8_layer.cu: one MoE layer whose expert weights and activations are 8-bit integers: routing by scores -> plan -> grouped gate|up (token rows gathered through
// xmap, bf16 out in sorted-row order) -> SiLU gate to 8-bit rows -> grouped down (bf16 rows scattered to token * topk + slot through ymap) -> combine in slot order.
// The two products leave bf16: their sums are exact, one rounding to 8 bits of mantissa is a sixteenth of a step of the 8-bit codes that follow, and f32 rows would double
// the traffic of the two passes that read them.
#include <math.h>
#include <stdlib.h>
#include "internal.h"
#include "mma_common.cuh"

namespace b200 {

// out[t] = sum over slots of w[t][s] * d[t * slots + s] in slot order, f32, bf16 rows in; a thread takes eight columns
__global__ void __launch_bounds__(256) combine16_kernel(uint32_t tokens, uint32_t slots, uint32_t hidden, const float *w, const uint16_t *d, float *__restrict__ out, uint16_t *__restrict__ out16) {
    griddep_chain();
    const uint32_t t = blockIdx.x;
    for (uint32_t c = threadIdx.x * 8u; c < hidden; c += 2048u) {
        float acc[8] = {};
        for (uint32_t s = 0; s < slots; s++) {
            const float ws = w[(size_t)t * slots + s];
            const uint4 v = *reinterpret_cast<const uint4 *>(d + ((size_t)t * slots + s) * hidden + c);
            const uint32_t b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                acc[2 * i] = fmaf(ws, __uint_as_float(b[i] << 16), acc[2 * i]);
                acc[2 * i + 1] = fmaf(ws, __uint_as_float(b[i] & 0xffff0000u), acc[2 * i + 1]);
            }
        }
        const size_t at = (size_t)t * hidden + c;
        if (out) { *reinterpret_cast<float4 *>(out + at) = make_float4(acc[0], acc[1], acc[2], acc[3]); *reinterpret_cast<float4 *>(out + at + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]); }
        if (out16) {
            uint4 o;
            o.x = bf16_rne_bits(acc[0]) | (bf16_rne_bits(acc[1]) << 16); o.y = bf16_rne_bits(acc[2]) | (bf16_rne_bits(acc[3]) << 16);
            o.z = bf16_rne_bits(acc[4]) | (bf16_rne_bits(acc[5]) << 16); o.w = bf16_rne_bits(acc[6]) | (bf16_rne_bits(acc[7]) << 16);
            *reinterpret_cast<uint4 *>(out16 + at) = o;
        }
    }
}

// sorted row p <- codes and scale of row xmap[p]: a warp per row, 16 bytes a lane. header: the plan's; one that was refused has no rows, and its maps are those of an earlier call
__global__ void __launch_bounds__(256) sort_rows_kernel(uint32_t rows, uint32_t k, const uint32_t *header, const uint32_t *xmap, const int8_t *q, const float *qs, int8_t *__restrict__ q_out, float *__restrict__ qs_out) {
    griddep_chain();
    const uint32_t lane = threadIdx.x & 31u, p = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (p >= min(rows, header[0])) return;
    const uint32_t src = xmap[p];
    const uint4 *from = reinterpret_cast<const uint4 *>(q + (size_t)src * k); uint4 *to = reinterpret_cast<uint4 *>(q_out + (size_t)p * k);
    for (uint32_t w0 = 0; w0 < k / 16u; w0 += 128u) {   // four independent 16-byte loads per lane before the first store
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) { const uint32_t w = w0 + lane + 32u * i; if (w < k / 16u) v[i] = from[w]; }
#pragma unroll
        for (int i = 0; i < 4; i++) { const uint32_t w = w0 + lane + 32u * i; if (w < k / 16u) to[w] = v[i]; }
    }
    if (lane == 0) qs_out[p] = qs[src];
}

constexpr int I8_REFUSED = 100;   // status of a refused plan: this and the plan's own word, as the FP8 layer reports it
static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace b200
using namespace b200;

struct OmegaGpuMoeI8Layer {
    const OmegaGpuI8Tensor *gu, *dn;     // not owned: experts x 2I rows of k = H; experts x H rows of k = I
    OmegaGpuMoeRouteConfig route;
    uint32_t hidden, inter, max_tokens, launches;
    char *base;
    float *bias, *wts, *xs, *ss, *as, *out32;   // ss, sq: input rows in sorted order
    int8_t *xq, *sq, *aq;
    uint16_t *logits, *x, *gu16, *dn16, *out16;
    uint32_t *ids, *counts, *starts, *xmap, *ymap, *tiles, *header, *scratch; size_t scratch_words;
};

namespace b200 {
// Rows per tile: room for an expert's average and half of it again while that is 32 or 64, so that most experts are one tile, which reads their weights once, and a tile leaves the
// pipeline its stages; above that the longest, in pairs of CTAs. Measured, 128 experts of 2048 x 768 with an uneven load, us with 64 / 96 / 128 / 256 rows: 512 tokens (32 an
// expert) 127 / 138 / 140 / 142, 768 tokens 143 / 150 / 150 / 151, 1024 tokens 163 / 161 / 158 / 158, 1500 tokens 195 / 196 / 179 / 176, 4096 tokens 436 / 412 / 320 / 290.
static uint32_t i8_tile_rows(uint32_t picks, uint32_t experts) {
    const uint32_t average = picks / experts;
    return average <= 21u ? 32u : average <= 56u ? 64u : 256u;
}
// Rows are copied into sorted order first where tiles are long: the product then fetches a tile's rows by TMA, which costs less than their copies through the
// map once a row is used by several channel blocks of a long tile. Measured: 512 tokens (32 rows an expert) 129.6 us unsorted, 133.7 sorted; gate|up alone of 4096 tokens
// 114 us and 14 for the copies against 199.
static bool i8_sorted(uint32_t picks, uint32_t experts) { return i8_tile_rows(picks, experts) == 256u; }
static uint32_t i8_max_tiles(uint32_t picks, uint32_t experts, uint32_t tile_rows) { return picks / tile_rows + (experts < picks ? experts : picks); }

static int i8_layer_run(OmegaGpuMoeI8Layer *L, uint32_t tokens, const uint16_t *logits, const int8_t *q, const float *qs, float *out32, uint16_t *out16, cudaStream_t s) {
    const uint32_t K = L->route.topk, E = L->route.experts, H = L->hidden, I = L->inter, R = tokens * K, tr = i8_tile_rows(R, E), most = i8_max_tiles(R, E, tr);
    OmegaGpuMoePlanOut o = {};
    o.counts_va = (uint64_t)(uintptr_t)L->counts; o.starts_va = (uint64_t)(uintptr_t)L->starts; o.xmap_va = (uint64_t)(uintptr_t)L->xmap; o.ymap_va = (uint64_t)(uintptr_t)L->ymap;
    o.tiles_va = (uint64_t)(uintptr_t)L->tiles; o.header_va = (uint64_t)(uintptr_t)L->header;
    I8Launch up = {}, dn = {};
    up.m = dn.m = most; up.tiles = dn.tiles = L->tiles; up.header = dn.header = L->header; up.tile_rows = dn.tile_rows = tr;
    const bool sorted = i8_sorted(R, E);
    up.n = 2u * I; up.x = sorted ? L->sq : q; up.xs = sorted ? L->ss : qs; up.x_rows = sorted ? R : tokens; up.xmap = sorted ? nullptr : L->xmap; up.y16 = L->gu16;   // sorted row p = x[xmap[p]] against its expert's 2I x H matrix
    dn.n = H; dn.x = L->aq; dn.xs = L->as; dn.x_rows = R; dn.ymap = L->ymap; dn.y16 = L->dn16;          // result of sorted row p to row ymap[p] = token * K + slot
    up.early = sorted; dn.early = 1;
    // one token's plan is its picks, and the routing writes it (25.8 -> 22.8 us for such a step)
    const bool ok = cuda_ok(launch_score_route(L->route, tokens, logits, 1, 0, L->bias, L->ids, L->wts, s, &o), "route launch") &&
                    (tokens == 1u || cuda_ok(launch_plan(tokens, K, E, K, tr, L->ids, o, s, L->scratch, L->scratch_words), "plan launch")) &&
                    (!sorted || cuda_ok(launch_chained(sort_rows_kernel, dim3((R + 7u) / 8u), dim3(256), 0, s, R, H, L->header, L->xmap, q, qs, L->sq, L->ss), "sort rows launch")) &&
                    cuda_ok(launch_i8_gemm(L->gu, up, s), "gate|up launch") &&
                    cuda_ok(launch_row_q8(R, I, 0, L->gu16, 1, 1, L->aq, L->as, s), "swiglu q8 launch") && cuda_ok(launch_i8_gemm(L->dn, dn, s), "down launch") &&
                    cuda_ok(launch_chained(combine16_kernel, dim3(tokens), dim3(H <= 1024u ? 128 : 256), 0, s, tokens, K, H, L->wts, L->dn16, out32, out16), "combine launch");
    L->launches = (sorted ? 6u : 5u) + (tokens == 1u ? 0u : plan_launch_count(R, E, L->scratch, L->scratch_words, o));
    return ok ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}
}  // namespace b200

extern "C" {

int omega_gpu_moe_i8_layer_create(const OmegaGpuI8Tensor *gate_up, const OmegaGpuI8Tensor *down, const OmegaGpuMoeRouteConfig *route, const float *bias, uint32_t max_tokens,
                                  OmegaGpuMoeI8Layer **out) {
    if (out) *out = nullptr;
    if (!out || !gate_up || !down || !max_tokens) return OMEGA_GPU_FP8_BAD_ARGS;
    const int rc = score_route_ok(route);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    const uint32_t E = route->experts, H = gate_up->k, I = down->k, K = route->topk;
    if (gate_up->n % E || down->n % E || gate_up->n / E != 2u * I || down->n / E != H) { set_error("i8 layer: gate|up must be experts x 2I rows of H columns and down experts x H rows of I columns"); return OMEGA_GPU_FP8_BAD_ARGS; }
    if (!q8_length_ok(H) || !q8_length_ok(I)) return OMEGA_GPU_FP8_BAD_ARGS;
    if ((uint64_t)max_tokens * K > (1u << 28)) return OMEGA_GPU_FP8_TOO_LARGE;
    if (bias) for (uint32_t e = 0; e < E; e++) if (bias[e] != bias[e]) { set_error("i8 layer: bias %u is NaN", e); return OMEGA_GPU_FP8_BAD_ARGS; }
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    OmegaGpuMoeI8Layer *L = (OmegaGpuMoeI8Layer *)calloc(1, sizeof *L);
    if (!L) return OMEGA_GPU_FP8_BAD_ARGS;
    L->gu = gate_up; L->dn = down; L->route = *route; L->hidden = H; L->inter = I; L->max_tokens = max_tokens;
    const size_t T = max_tokens, R = T * K;
    L->scratch_words = plan_scratch_words((uint32_t)R, E);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return o; };
    const size_t o_b = take((size_t)E * 4), o_lg = take(T * E * 2), o_x = take(T * H * 2), o_xq = take(T * H), o_xs = take(T * 4), o_sq = take(i8_sorted((uint32_t)R, E) ? R * H : 0), o_ss = take(i8_sorted((uint32_t)R, E) ? R * 4 : 0), o_ids = take(R * 4), o_wts = take(R * 4), o_cnt = take((size_t)E * 4),
                 o_st = take((size_t)E * 4), o_xm = take((R + 8) * 4), o_ym = take((R + 8) * 4), o_tl = take((R + E) * 16), o_hdr = take(64), o_sc = take(L->scratch_words * 4),
                 o_gu = take(R * 2 * I * 2), o_aq = take(R * I), o_as = take(R * 4), o_dn = take(R * H * 2), o_o32 = take(T * H * 4), o_o16 = take(T * H * 2);
    if (!cuda_ok(cudaMalloc(&L->base, off), "cudaMalloc(i8 layer)") || !cuda_ok(cudaMemset(L->base, 0, off), "memset") ||
        (bias && !cuda_ok(cudaMemcpy(L->base + o_b, bias, (size_t)E * 4, cudaMemcpyHostToDevice), "copy bias")) || !cuda_ok(cudaDeviceSynchronize(), "i8 layer")) {
        if (L->base) cudaFree(L->base);
        free(L);
        return OMEGA_GPU_FP8_CHIP_FAIL;
    }
    char *b = L->base;
    L->bias = bias ? (float *)(b + o_b) : nullptr; L->logits = (uint16_t *)(b + o_lg); L->x = (uint16_t *)(b + o_x); L->xq = (int8_t *)(b + o_xq); L->xs = (float *)(b + o_xs);
    L->sq = (int8_t *)(b + o_sq); L->ss = (float *)(b + o_ss); L->ids = (uint32_t *)(b + o_ids); L->wts = (float *)(b + o_wts); L->counts = (uint32_t *)(b + o_cnt); L->starts = (uint32_t *)(b + o_st); L->xmap = (uint32_t *)(b + o_xm);
    L->ymap = (uint32_t *)(b + o_ym); L->tiles = (uint32_t *)(b + o_tl); L->header = (uint32_t *)(b + o_hdr); L->scratch = (uint32_t *)(b + o_sc); L->gu16 = (uint16_t *)(b + o_gu);
    L->aq = (int8_t *)(b + o_aq); L->as = (float *)(b + o_as); L->dn16 = (uint16_t *)(b + o_dn); L->out32 = (float *)(b + o_o32); L->out16 = (uint16_t *)(b + o_o16);
    *out = L;
    return OMEGA_GPU_FP8_OK;
}

void omega_gpu_moe_i8_layer_free(OmegaGpuMoeI8Layer *L) {
    if (!L) return;
    Lock l;
    if (L->base) cudaFree(L->base);
    free(L);
}

int omega_gpu_moe_i8_layer_q8_async(OmegaGpuMoeI8Layer *L, uint32_t tokens, uint64_t logits_va, uint64_t q_va, uint64_t s_va, uint64_t out_f32_va, uint64_t out_bf16_va, void *stream) {
    if (!L || !tokens || !logits_va || !q_va || !s_va || (!out_f32_va && !out_bf16_va) || ((q_va | out_f32_va | out_bf16_va) & 15u) || (s_va & 3u) || (logits_va & 1u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > L->max_tokens) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return i8_layer_run(L, tokens, (const uint16_t *)(uintptr_t)logits_va, (const int8_t *)(uintptr_t)q_va, (const float *)(uintptr_t)s_va, (float *)(uintptr_t)out_f32_va,
                        (uint16_t *)(uintptr_t)out_bf16_va, (cudaStream_t)stream);
}

int omega_gpu_moe_i8_layer_async(OmegaGpuMoeI8Layer *L, uint32_t tokens, uint64_t logits_va, uint64_t x_va, uint64_t out_f32_va, uint64_t out_bf16_va, void *stream) {
    if (!L || !tokens || !logits_va || !x_va || (!out_f32_va && !out_bf16_va) || ((x_va | out_f32_va | out_bf16_va) & 15u) || (logits_va & 1u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > L->max_tokens) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    cudaStream_t s = (cudaStream_t)stream;
    if (!cuda_ok(launch_row_q8(tokens, L->hidden, 0, (const void *)(uintptr_t)x_va, 1, 0, L->xq, L->xs, s), "quant q8 launch")) return OMEGA_GPU_FP8_CHIP_FAIL;
    const int rc = i8_layer_run(L, tokens, (const uint16_t *)(uintptr_t)logits_va, L->xq, L->xs, (float *)(uintptr_t)out_f32_va, (uint16_t *)(uintptr_t)out_bf16_va, s);
    L->launches++;
    return rc;
}

int omega_gpu_moe_i8_layer_bf16(OmegaGpuMoeI8Layer *L, uint32_t tokens, const uint16_t *logits_bf16, const uint16_t *x_bf16, uint16_t *out_bf16, float *out_f32, uint32_t *ids, float *wts) {
    if (!L || !tokens || !logits_bf16 || !x_bf16 || (!out_bf16 && !out_f32)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > L->max_tokens) return OMEGA_GPU_FP8_TOO_LARGE;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    cudaStream_t s = st().stream;
    const size_t xb = (size_t)tokens * L->hidden * 2, rb = (size_t)tokens * L->route.topk * 4;
    if (!to_device(L->logits, logits_bf16, (size_t)tokens * L->route.experts * 2, s) || !to_device(L->x, x_bf16, xb, s)) return OMEGA_GPU_FP8_CHIP_FAIL;
    const int rc = omega_gpu_moe_i8_layer_async(L, tokens, (uint64_t)(uintptr_t)L->logits, (uint64_t)(uintptr_t)L->x, (uint64_t)(uintptr_t)L->out32, (uint64_t)(uintptr_t)L->out16, s);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    bool ok = true;
    if (out_bf16) ok = ok && to_host(out_bf16, L->out16, xb, s);
    if (out_f32) ok = ok && to_host(out_f32, L->out32, xb * 2, s);
    if (ids) ok = ok && to_host(ids, L->ids, rb, s);
    if (wts) ok = ok && to_host(wts, L->wts, rb, s);
    if (!ok) return OMEGA_GPU_FP8_CHIP_FAIL;
    const int status = omega_gpu_moe_i8_layer_status(L, s);
    if (status > I8_REFUSED) { set_error("i8 layer: routing plan refused (status %d)", status - I8_REFUSED); return OMEGA_GPU_FP8_BAD_ARGS; }
    return status == 0 ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_moe_i8_layer_status(OmegaGpuMoeI8Layer *L, void *stream) {
    if (!L) return OMEGA_GPU_FP8_BAD_ARGS;
    Lock l;
    cudaStream_t s = (cudaStream_t)stream;
    uint32_t refused = 0;
    if (!cuda_ok(cudaMemcpyAsync(&refused, L->header + 3, 4, cudaMemcpyDeviceToHost, s), "copy status")) return OMEGA_GPU_FP8_CHIP_FAIL;
    const int up = i8_status(L->gu, s), down = up ? 0 : i8_status(L->dn, s);   // they wait for s
    return up ? up : down ? down : refused ? I8_REFUSED + (int)refused : 0;
}

uint32_t omega_gpu_moe_i8_layer_launches(const OmegaGpuMoeI8Layer *L) { return L ? L->launches : 0; }

}  // extern "C"
