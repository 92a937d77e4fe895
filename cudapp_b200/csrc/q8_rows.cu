// q8_rows.cu: rows of signed 8-bit codes with one f32 scale each, the activations of the 8-bit integer product (i8_gemm.cu): from residual + RMSNorm, from a SiLU
// gate, or from rows as they are.
//
//   s = max(max |y|, 2^-100) / 127,  q = round-to-nearest-even(y / s) in -127 .. 127;  a row with a NaN or an infinity: q = 0, s = NaN.
//
// All three read each input once: a row stays in registers between the reduction and the codes (V groups of 8 values a thread), so they are bound by memory
// for many rows (norm of 4096 x 2048 f32: 18.8 us of 17.0 at the copy rate; gate of 32768 x 768 bf16: 21.5 us of 19.6, 31 with a CTA per eight rows, no row requested ahead
// and conversion instructions for the codes) and by one load and one reduction for few (1.9 us). Largest values are reduced as the bits of |y|: NaN lies above infinity there and is not lost, as fmaxf loses it.
#include <math.h>
#include "internal.h"
#include "mma_common.cuh"

namespace b200 {

constexpr uint32_t Q8_INF = 0x7f800000u, Q8_MOST = 16384, Q8_MOST_ROWS = 1u << 30;

__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u); v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
    v[4] = __uint_as_float(w.z << 16); v[5] = __uint_as_float(w.z & 0xffff0000u); v[6] = __uint_as_float(w.w << 16); v[7] = __uint_as_float(w.w & 0xffff0000u);
}
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// the row's scale from the bits of its largest |y|; inv = 1 / scale, 0 for a row that is not finite
__device__ __forceinline__ float q8_scale(uint32_t top, float *inv) {
    const float m = fmaxf(__uint_as_float(top), 7.888609052210118e-31f /* 2^-100 */), s = __fdiv_rn(m, 127.0f);
    const bool fine = top < Q8_INF;
    *inv = fine ? __fdiv_rn(127.0f, m) : 0.0f;
    return fine ? s : __uint_as_float(0x7fffffffu);
}
// Codes of eight values: y * (127 / max) is within two roundings of y / s, so a code differs from the quotient's only next to a border between two codes. Adding 1.5 * 2^23
// leaves the rounded value in the low bits of the sum: |y * inv| < 127.0001, and the conversion instructions share the exponential's slow unit.
__device__ __forceinline__ uint2 q8_pack(const float (&y)[8], float inv, bool fine) {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = __float_as_uint(fmaf(y[i], inv, 12582912.0f));
    uint2 o;
    o.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    return fine ? o : make_uint2(0, 0);
}

// ------------------------------------------------------------------ residual + RMSNorm
// One CTA of W warps per token. Sum of squares in binary64, as residual_norm_kernel's; max |h * w| is reduced in the same exchange and multiplied by the
// norm's factor afterwards, so there is one barrier between the loads and the codes.
template <int W, int V, typename X, typename M>
__global__ void __launch_bounds__(W * 32) norm_q8_kernel(uint32_t hidden, float eps, const X *x, const M *m, float *h_out, const float *norm_w, uint16_t *xn, int8_t *__restrict__ q, float *__restrict__ s) {
    griddep_chain();
    __shared__ double r_sq[W];
    __shared__ uint32_t r_top[W];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const size_t row = (size_t)blockIdx.x * hidden;
    float h[V][8];
    double sq = 0.0; uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t c = (i * W * 32u + tid) * 8u;
        if (c < hidden) {
            load8(x + row + c, h[i]);
            if (m) {
                float d[8]; load8(m + row + c, d);
#pragma unroll
                for (int j = 0; j < 8; j++) h[i][j] = __fadd_rn(h[i][j], d[j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t c = (i * W * 32u + tid) * 8u;
        if (c >= hidden) continue;
        if (h_out) { *reinterpret_cast<float4 *>(h_out + row + c) = make_float4(h[i][0], h[i][1], h[i][2], h[i][3]); *reinterpret_cast<float4 *>(h_out + row + c + 4) = make_float4(h[i][4], h[i][5], h[i][6], h[i][7]); }
        float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (norm_w) load8(norm_w + c, w);
#pragma unroll
        for (int j = 0; j < 8; j++) { sq += (double)h[i][j] * (double)h[i][j]; h[i][j] *= w[j]; top = max(top, abs_bits(h[i][j])); }
    }
    for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) { r_sq[warp] = sq; r_top[warp] = top; }
    __syncthreads();
    double a = 0.0;
#pragma unroll
    for (int i = 0; i < W; i++) { a += r_sq[i]; top = max(top, r_top[i]); }
    const double rms = sqrt(a / (double)hidden + (double)eps);
    // keeps the factor of huge rows out of the subnormal numbers and that of tiny ones (no eps) out of the infinite ones
    const float pre = rms > 1.2676506002282294e30 /* 2^100 */ ? 5.421010862427522e-20f /* 2^-64 */ : rms < 7.888609052210118e-31 /* 2^-100 */ ? 1.8446744073709552e19f /* 2^64 */ : 1.0f;
    const float r = (float)(1.0 / (rms * (double)pre));
    // a row that is not finite has a NaN or an infinity among the h * w (0 * infinity is NaN)
    const uint32_t y_top = top < Q8_INF ? abs_bits(__uint_as_float(top) * pre * r) : Q8_INF;
    float inv; const float sc = q8_scale(y_top, &inv);
    const bool fine = y_top < Q8_INF;
    if (tid == 0) s[blockIdx.x] = sc;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t c = (i * W * 32u + tid) * 8u;
        if (c >= hidden) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = h[i][j] * pre * r;
        *reinterpret_cast<uint2 *>(q + row + c) = q8_pack(h[i], inv, fine);
        if (xn) {
            uint4 o;
            o.x = bf16_rne_bits(h[i][0]) | (bf16_rne_bits(h[i][1]) << 16); o.y = bf16_rne_bits(h[i][2]) | (bf16_rne_bits(h[i][3]) << 16);
            o.z = bf16_rne_bits(h[i][4]) | (bf16_rne_bits(h[i][5]) << 16); o.w = bf16_rne_bits(h[i][6]) | (bf16_rne_bits(h[i][7]) << 16);
            *reinterpret_cast<uint4 *>(xn + row + c) = o;
        }
    }
}

// ------------------------------------------------------------------ rows as they are, or silu(gate) * up
// W warps per row; with W = 1 a CTA holds eight rows at a time. A worker takes every so-manieth row and requests the next one's values before it computes with this one's.
template <typename X> struct Raw8;
template <> struct Raw8<uint16_t> {
    uint4 w;
    __device__ __forceinline__ void load(const uint16_t *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u); v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
        v[4] = __uint_as_float(w.z << 16); v[5] = __uint_as_float(w.z & 0xffff0000u); v[6] = __uint_as_float(w.w << 16); v[7] = __uint_as_float(w.w & 0xffff0000u);
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) { a = *reinterpret_cast<const float4 *>(p); b = *reinterpret_cast<const float4 *>(p + 4); }
    __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
};
template <int W, int V, bool GATE, typename X>
__global__ void __launch_bounds__(256) row_q8_kernel(uint32_t rows, uint32_t n, size_t stride, const X *x, int8_t *__restrict__ q, float *__restrict__ s) {
    griddep_chain();
    __shared__ uint32_t r_top[2][8];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, tid = W == 1 ? lane : threadIdx.x, step = W == 1 ? gridDim.x * 8u : gridDim.x;
    Raw8<X> g[V], u[GATE ? V : 1];
    auto fetch = [&](uint32_t r) {
        const X *p = reinterpret_cast<const X *>(reinterpret_cast<const uint8_t *>(x) + (size_t)r * stride);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (i * W * 32u + tid) * 8u;
            if (c < n) { g[i].load(p + c); if constexpr (GATE) u[i].load(p + n + c); }
        }
    };
    uint32_t r = W == 1 ? blockIdx.x * 8u + warp : blockIdx.x, turn = 0;
    if (r < rows) fetch(r);
    for (; r < rows; r += step, turn ^= 1u) {   // W > 1: the same rows for the whole CTA
        float y[V][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (i * W * 32u + tid) * 8u;
            if (c >= n) continue;
            g[i].get(y[i]);
            if constexpr (GATE) {
                float v[8]; u[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; j++) y[i][j] = silu_mul_dev(y[i][j], v[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) top = max(top, abs_bits(y[i][j]));
        }
        if (r + step < rows) fetch(r + step);
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (W > 1) {
            if (lane == 0) r_top[turn][warp] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < W; i++) top = max(top, r_top[turn][i]);
        }
        float inv; const float sc = q8_scale(top, &inv);
        const bool fine = top < Q8_INF;
        if (tid == 0) s[r] = sc;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (i * W * 32u + tid) * 8u;
            if (c < n) *reinterpret_cast<uint2 *>(q + (size_t)r * n + c) = q8_pack(y[i], inv, fine);
        }
    }
}

template <typename X, typename M>
static cudaError_t norm_launch(uint32_t tokens, uint32_t hidden, float eps, const X *x, const M *m, float *h, const float *nw, uint16_t *xn, int8_t *q, float *s, cudaStream_t st_) {
#define NORM(WV, VV) return launch_chained(norm_q8_kernel<WV, VV, X, M>, dim3(tokens), dim3((WV) * 32), 0, st_, hidden, eps, x, m, h, nw, xn, q, s)
    if (hidden <= 512) NORM(2, 1);
    if (hidden <= 2048) NORM(8, 1);
    if (hidden <= 4096) NORM(8, 2);
    if (hidden <= 8192) NORM(8, 4);
    NORM(8, 8);
#undef NORM
}
cudaError_t launch_norm_q8(uint32_t tokens, uint32_t hidden, float eps, const void *x, int x_bf16, const void *m, int m_bf16, float *h, const float *nw, uint16_t *xn, int8_t *q, float *s, cudaStream_t st_) {
    if (x_bf16) return m_bf16 ? norm_launch(tokens, hidden, eps, (const uint16_t *)x, (const uint16_t *)m, h, nw, xn, q, s, st_) : norm_launch(tokens, hidden, eps, (const uint16_t *)x, (const float *)m, h, nw, xn, q, s, st_);
    return m_bf16 ? norm_launch(tokens, hidden, eps, (const float *)x, (const uint16_t *)m, h, nw, xn, q, s, st_) : norm_launch(tokens, hidden, eps, (const float *)x, (const float *)m, h, nw, xn, q, s, st_);
}
template <bool GATE, typename X>
static cudaError_t row_launch(uint32_t rows, uint32_t n, size_t stride, const X *x, int8_t *q, float *s, cudaStream_t st_) {
    // Four CTAs an SM: by its registers the gate of bf16 rows up to 768 columns has as many resident, forms with fewer values a thread up to eight, those with more one to three;
    // of these the CTAs that do not fit start as others end, and only then request their first row
    const uint32_t most = 4u * (uint32_t)(st().sm_count ? st().sm_count : 148);
#define ROW(WV, VV) { const uint32_t ctas = (WV) == 1 ? (rows + 7) / 8 : rows; return launch_chained(row_q8_kernel<WV, VV, GATE, X>, dim3(ctas < most ? ctas : most), dim3(256), 0, st_, rows, n, stride, x, q, s); }
    if (n <= 256) ROW(1, 1);
    if (n <= 512) ROW(1, 2);
    if (n <= 768) ROW(1, 3);
    if (n <= 1024) ROW(1, 4);
    if (n <= 2048) ROW(8, 1);
    if (n <= 4096) ROW(8, 2);
    if (n <= 8192) ROW(8, 4);
    ROW(8, 8);
#undef ROW
}
cudaError_t launch_row_q8(uint32_t rows, uint32_t n, size_t stride, const void *x, int x_bf16, int gate, int8_t *q, float *s, cudaStream_t st_) {
    if (!stride) stride = (size_t)n * (gate ? 2 : 1) * (x_bf16 ? 2 : 4);
    if (gate) return x_bf16 ? row_launch<true>(rows, n, stride, (const uint16_t *)x, q, s, st_) : row_launch<true>(rows, n, stride, (const float *)x, q, s, st_);
    return x_bf16 ? row_launch<false>(rows, n, stride, (const uint16_t *)x, q, s, st_) : row_launch<false>(rows, n, stride, (const float *)x, q, s, st_);
}
bool q8_length_ok(uint32_t n) {
    if (n && n % 16u == 0 && n <= Q8_MOST) return true;
    set_error("8-bit rows: length %u is no multiple of 16 up to %u", n, Q8_MOST);
    return false;
}

}  // namespace b200
using namespace b200;

extern "C" {

int omega_gpu_residual_norm_q8_async(uint32_t tokens, uint32_t hidden, float eps, uint64_t x16_va, uint64_t m_va, int m_bf16, uint64_t h_in_va, uint64_t h_va,
                                     uint64_t norm_w_va, uint64_t xn_bf16_va, uint64_t q_va, uint64_t s_va, void *stream) {
    if (!tokens || !x16_va == !h_in_va || !q_va || !s_va || !(eps >= 0.0f) || ((x16_va | m_va | h_in_va | h_va | norm_w_va | xn_bf16_va | q_va) & 15u) || (s_va & 3u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (!q8_length_ok(hidden)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > Q8_MOST_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return cuda_ok(launch_norm_q8(tokens, hidden, eps, (const void *)(uintptr_t)(x16_va ? x16_va : h_in_va), x16_va != 0, (const void *)(uintptr_t)m_va, m_bf16 != 0, (float *)(uintptr_t)h_va,
                                  (const float *)(uintptr_t)norm_w_va, (uint16_t *)(uintptr_t)xn_bf16_va, (int8_t *)(uintptr_t)q_va, (float *)(uintptr_t)s_va, (cudaStream_t)stream), "norm q8 launch")
               ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_quant_q8_async(uint32_t rows, uint32_t k, uint64_t x_va, int x_bf16, uint32_t x_stride_bytes, uint64_t q_va, uint64_t s_va, void *stream) {
    if (!rows || !x_va || !q_va || !s_va || ((x_va | q_va | x_stride_bytes) & 15u) || (s_va & 3u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (!q8_length_ok(k) || (x_stride_bytes && x_stride_bytes < k * (x_bf16 ? 2u : 4u))) return OMEGA_GPU_FP8_BAD_ARGS;
    if (rows > Q8_MOST_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return cuda_ok(launch_row_q8(rows, k, x_stride_bytes, (const void *)(uintptr_t)x_va, x_bf16 != 0, 0, (int8_t *)(uintptr_t)q_va, (float *)(uintptr_t)s_va, (cudaStream_t)stream), "quant q8 launch")
               ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_swiglu_q8_async(uint32_t rows, uint32_t inter, uint64_t gu_va, int gu_bf16, uint64_t q_va, uint64_t s_va, void *stream) {
    if (!rows || !gu_va || !q_va || !s_va || ((gu_va | q_va) & 15u) || (s_va & 3u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (!q8_length_ok(inter)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (rows > Q8_MOST_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    return cuda_ok(launch_row_q8(rows, inter, 0, (const void *)(uintptr_t)gu_va, gu_bf16 != 0, 1, (int8_t *)(uintptr_t)q_va, (float *)(uintptr_t)s_va, (cudaStream_t)stream), "swiglu q8 launch")
               ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_residual_norm_q8_f32(uint32_t tokens, uint32_t hidden, float eps, const float *x, const float *m, const float *norm_w, float *h, int8_t *q, float *sc) {
    if (!tokens || !x || !q || !sc || !(eps >= 0.0f) || !q8_length_ok(hidden)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (tokens > Q8_MOST_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    const size_t qb = (size_t)tokens * hidden, xb = qb * 4, wb = (size_t)hidden * 4, sb = (size_t)tokens * 4;
    float *dx = (float *)stage(0, xb), *dm = (float *)stage(1, xb), *dw = (float *)stage(2, wb + sb); int8_t *dq = (int8_t *)stage(3, qb);
    if (!dx || !dm || !dw || !dq) return OMEGA_GPU_FP8_CHIP_FAIL;
    float *ds = dw + hidden;
    cudaStream_t s = st().stream;
    const bool ok = to_device(dx, x, xb, s) && (!m || to_device(dm, m, xb, s)) && (!norm_w || to_device(dw, norm_w, wb, s)) &&
                    cuda_ok(launch_norm_q8(tokens, hidden, eps, dx, 0, m ? dm : nullptr, 0, dx, norm_w ? dw : nullptr, nullptr, dq, ds, s), "norm q8 launch") &&
                    to_host(q, dq, qb, s) && to_host(sc, ds, sb, s) && (!h || to_host(h, dx, xb, s)) && cuda_ok(cudaStreamSynchronize(s), "norm q8");
    return ok ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_swiglu_q8_f32(uint32_t rows, uint32_t inter, const float *gu, int8_t *q, float *sc) {
    if (!rows || !gu || !q || !sc || !q8_length_ok(inter)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (rows > Q8_MOST_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    const size_t qb = (size_t)rows * inter, gb = qb * 8, sb = (size_t)rows * 4;
    float *dg = (float *)stage(0, gb), *ds = (float *)stage(2, sb); int8_t *dq = (int8_t *)stage(1, qb);
    if (!dg || !dq || !ds) return OMEGA_GPU_FP8_CHIP_FAIL;
    cudaStream_t s = st().stream;
    const bool ok = to_device(dg, gu, gb, s) && cuda_ok(launch_row_q8(rows, inter, 0, dg, 0, 1, dq, ds, s), "swiglu q8 launch") && to_host(q, dq, qb, s) && to_host(sc, ds, sb, s) &&
                    cuda_ok(cudaStreamSynchronize(s), "swiglu q8");
    return ok ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

}  // extern "C"
