// i8_gemm.cu: products of signed 8-bit rows with signed 8-bit weights, one f32 scale per row and per weight row.
//
//   y[i][j] = (sum over c of x[i][c] w[j][c]) * (xs[i] ws[j]),  the sum in 32-bit integers: exact for k <= 32768, whatever the order it is taken in.
//
// Weights are the tensor-core operation's M operand and activation rows its N operand, so a few rows (decode) waste no part of a tile.
#include <math.h>
#include <stdlib.h>
#include "internal.h"
#include "mma_common.cuh"

namespace b200 {

constexpr uint32_t I8_MAX_K = 32768, I8_MAX_ROWS = 1u << 30;   // rows: of weights and of one call; row numbers are signed in tensor maps

struct I8Args {
    const int8_t *w, *x; const float *ws, *xs; uint16_t *y16; float *y32;
    size_t x_stride; uint32_t m, n, k;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A few dense rows: a CTA takes 16 channels and all 8 NT activation rows, its eight warps take turns of 128 columns and add their sums up in shared memory. Operands go from
// memory straight into the fragments: the sum over k may be taken in any order, so a lane's 16 consecutive bytes serve as its parts of two products. Bound by the weights'
// way from memory: a warp requests those of four turns (4096 columns of the CTA's 16 channels, 64 KB) before it uses the first, and before the kernels ahead in the
// stream have completed. 1 x 4096 x 4096: 2.9 us, 5.7 TB/s; 16 rows 3.8, 32 rows 5.6 (7.2 on tcgen05, whose set-up and exchange these sizes do not earn back).
template <int NT>
__global__ void __launch_bounds__(256, 2) i8_rows_kernel(const I8Args a) {
    __shared__ int red[8][16][8 * NT + 1];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3u, n0 = blockIdx.x * 16u;
    const int8_t *w0 = a.w + (size_t)min(n0 + g, a.n - 1u) * a.k, *w1 = a.w + (size_t)min(n0 + g + 8u, a.n - 1u) * a.k;
    int acc[NT][4] = {};
    for (uint32_t c0 = warp * 128u; c0 < a.k || c0 < 1024u; c0 += 4096u) {   // once for every warp: it has to come to the wait
        uint4 u[8], v[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t c = c0 + (i >> 1) * 1024u + (i & 1u) * 64u + t * 16u;
            u[i] = v[i] = make_uint4(0, 0, 0, 0);
            if (c < a.k) { u[i] = __ldg(reinterpret_cast<const uint4 *>(w0 + c)); v[i] = __ldg(reinterpret_cast<const uint4 *>(w1 + c)); }
        }
        if (c0 < 1024u) griddep_chain();
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t c = c0 + (i >> 1) * 1024u + (i & 1u) * 64u + t * 16u;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const uint32_t r = j * 8u + g;
                uint4 b = make_uint4(0, 0, 0, 0);
                if (r < a.m && c < a.k) b = *reinterpret_cast<const uint4 *>(a.x + (size_t)r * a.x_stride + c);
                mma_s8(acc[j], u[i].x, v[i].x, u[i].y, v[i].y, b.x, b.y);
                mma_s8(acc[j], u[i].z, v[i].z, u[i].w, v[i].w, b.z, b.w);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        red[warp][g][j * 8 + 2 * t] = acc[j][0]; red[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
        red[warp][g + 8][j * 8 + 2 * t] = acc[j][2]; red[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 128u * NT; i += 256u) {
        const uint32_t ch = i & 15u, r = i >> 4, n = n0 + ch;
        if (r >= a.m || n >= a.n) continue;
        int sum = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) sum += red[q][ch][r];
        const float y = (float)sum * (a.xs[r] * __ldg(a.ws + n));
        const size_t at = (size_t)r * a.n + n;
        if (a.y32) a.y32[at] = y;
        if (a.y16) a.y16[at] = (uint16_t)bf16_rne_bits(y);
    }
}

cudaError_t launch_i8_gemm(const OmegaGpuI8Tensor *t, const I8Launch &l, cudaStream_t s) {
    // Few rows go to the kernel above while its CTAs are resident at once, and up to 8 in any case (8192 x 8192: 8 rows 16.0 us here, 32 rows 23.9 here and 15.3 there). An expert's
    // few rows do not: a layer's gate|up of 64 tokens takes 82 us here and 50 there, its whole step of one token 29 and 26.
    const uint32_t blocks = (l.n + 15u) / 16u, sms = st().sm_count ? st().sm_count : 148;
    if (l.tiles || l.m > 32u || (l.m > 8u && blocks > 2u * sms)) return launch_i8_mma(t, l, s);
    I8Args a = {};
    a.w = t->w; a.ws = t->s; a.x = l.x; a.xs = l.xs; a.y16 = l.y16; a.y32 = l.y32; a.x_stride = l.x_stride ? l.x_stride : t->k; a.m = l.m; a.n = l.n; a.k = t->k;
    const dim3 grid(blocks), block(256);
    return l.m <= 8u ? launch_chained(i8_rows_kernel<1>, grid, block, 0, s, a) : l.m <= 16u ? launch_chained(i8_rows_kernel<2>, grid, block, 0, s, a)
         : l.m <= 24u ? launch_chained(i8_rows_kernel<3>, grid, block, 0, s, a) : launch_chained(i8_rows_kernel<4>, grid, block, 0, s, a);
}

int i8_status(const OmegaGpuI8Tensor *t, cudaStream_t s) {
    uint32_t code = 0;
    if (!cuda_ok(cudaMemcpyAsync(&code, t->err, 4, cudaMemcpyDeviceToHost, s), "copy i8 status") || !cuda_ok(cudaStreamSynchronize(s), "i8 status")) return OMEGA_GPU_FP8_CHIP_FAIL;
    if (code) { set_error("i8 product: a bounded wait inside the tensor-core kernel ran out (code %u)", code); st().latched = true; }
    return (int)code;
}

}  // namespace b200
using namespace b200;

extern "C" {

static int i8_shape(uint32_t n, uint32_t k) {
    if (!n || !k || k % 16u) return OMEGA_GPU_FP8_BAD_ARGS;
    return k > I8_MAX_K || n > I8_MAX_ROWS ? OMEGA_GPU_FP8_TOO_LARGE : OMEGA_GPU_FP8_OK;
}
static int i8_scales(const float *s, uint32_t n) {
    for (uint32_t i = 0; i < n; i++) {
        if (s[i] != s[i]) { set_error("i8 upload: scale %u is NaN", i); return OMEGA_GPU_FP8_NAN_WEIGHT; }
        if (fabsf(s[i]) > 3.0e38f) { set_error("i8 upload: scale %u is infinite or overflowing", i); return OMEGA_GPU_FP8_BAD_ARGS; }
    }
    return OMEGA_GPU_FP8_OK;
}
static int i8_make(uint32_t n, uint32_t k, const void *w, const void *scale, cudaMemcpyKind kind, OmegaGpuI8Tensor **out) {
    OmegaGpuI8Tensor *t = (OmegaGpuI8Tensor *)calloc(1, sizeof *t);
    if (!t) return OMEGA_GPU_FP8_BAD_ARGS;
    t->n = n; t->k = k;
    cudaStream_t s = st().stream;
    const bool ok = cuda_ok(cudaMalloc(&t->w, (size_t)n * k), "cudaMalloc(i8)") && cuda_ok(cudaMalloc(&t->s, (size_t)n * 4 + 16), "cudaMalloc(i8 scales)") &&
                    cuda_ok(cudaMemsetAsync(t->s, 0, (size_t)n * 4 + 16, s), "memset") &&
                    cuda_ok(cudaMemcpyAsync(t->w, w, (size_t)n * k, kind, s), "copy i8") && cuda_ok(cudaMemcpyAsync(t->s, scale, (size_t)n * 4, kind, s), "copy i8 scales") &&
                    cuda_ok(cudaStreamSynchronize(s), "i8 upload");
    if (!ok) { if (t->w) cudaFree(t->w); if (t->s) cudaFree(t->s); free(t); return OMEGA_GPU_FP8_CHIP_FAIL; }
    t->err = reinterpret_cast<uint32_t *>(t->s + n);
    *out = t;
    return OMEGA_GPU_FP8_OK;
}

int omega_gpu_i8_upload(uint32_t n, uint32_t k, const int8_t *w, const float *scale, OmegaGpuI8Tensor **out) {
    if (out) *out = nullptr;
    if (!out || !w || !scale) return OMEGA_GPU_FP8_BAD_ARGS;
    int rc = i8_shape(n, k);
    if (rc == OMEGA_GPU_FP8_OK) rc = i8_scales(scale, n);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    return i8_make(n, k, w, scale, cudaMemcpyHostToDevice, out);
}

int omega_gpu_i8_upload_dev(uint32_t n, uint32_t k, uint64_t w_va, uint64_t scale_va, OmegaGpuI8Tensor **out) {
    if (out) *out = nullptr;
    if (!out || !w_va || !scale_va) return OMEGA_GPU_FP8_BAD_ARGS;
    int rc = i8_shape(n, k);
    if (rc != OMEGA_GPU_FP8_OK) return rc;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    float *h = (float *)malloc((size_t)n * 4);
    if (!h) return OMEGA_GPU_FP8_BAD_ARGS;
    rc = cuda_ok(cudaDeviceSynchronize(), "sync before upload") &&   // the caller's producer kernels may run on another stream
                 cuda_ok(cudaMemcpy(h, (const void *)(uintptr_t)scale_va, (size_t)n * 4, cudaMemcpyDeviceToHost), "copy i8 scales") ? i8_scales(h, n) : OMEGA_GPU_FP8_CHIP_FAIL;
    free(h);
    return rc == OMEGA_GPU_FP8_OK ? i8_make(n, k, (const void *)(uintptr_t)w_va, (const void *)(uintptr_t)scale_va, cudaMemcpyDeviceToDevice, out) : rc;
}

void omega_gpu_i8_free(OmegaGpuI8Tensor *t) {
    if (!t) return;
    Lock l;
    if (t->w) cudaFree(t->w);
    if (t->s) cudaFree(t->s);
    free(t);
}

int omega_gpu_i8_gemm_async(const OmegaGpuI8Tensor *t, uint32_t m, uint64_t x_va, uint32_t x_stride_bytes, uint64_t x_scale_va, uint64_t y_bf16_va, uint64_t y_f32_va, void *stream) {
    if (!t || !m || !x_va || !x_scale_va || (!y_bf16_va && !y_f32_va) || ((x_va | x_stride_bytes | y_bf16_va | y_f32_va) & 15u) || (x_scale_va & 3u)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (m > I8_MAX_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    if (x_stride_bytes && x_stride_bytes < t->k) { set_error("i8 gemm: rows of %u bytes %u bytes apart", t->k, x_stride_bytes); return OMEGA_GPU_FP8_BAD_ARGS; }
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    I8Launch a = {};
    a.m = m; a.n = t->n; a.x = (const int8_t *)(uintptr_t)x_va; a.x_stride = x_stride_bytes; a.x_rows = m; a.xs = (const float *)(uintptr_t)x_scale_va;
    a.y16 = (uint16_t *)(uintptr_t)y_bf16_va; a.y32 = (float *)(uintptr_t)y_f32_va;
    return cuda_ok(launch_i8_gemm(t, a, (cudaStream_t)stream), "i8 gemm launch") ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_i8_gemm(const OmegaGpuI8Tensor *t, uint32_t m, const int8_t *x, const float *x_scale, uint16_t *y16, float *y32) {
    if (!t || !m || !x || !x_scale || (!y16 && !y32)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (m > I8_MAX_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    Lock l;
    if (!dev_open()) return OMEGA_GPU_FP8_CHIP_FAIL;
    const size_t xb = (size_t)m * t->k, yb = (size_t)m * t->n;
    int8_t *dx = (int8_t *)stage(0, xb); uint16_t *d16 = y16 ? (uint16_t *)stage(1, yb * 2) : nullptr; float *d32 = y32 ? (float *)stage(2, yb * 4) : nullptr, *ds = (float *)stage(3, (size_t)m * 4);
    if (!dx || !ds || (y16 && !d16) || (y32 && !d32)) return OMEGA_GPU_FP8_CHIP_FAIL;
    cudaStream_t s = st().stream;
    I8Launch a = {};
    a.m = m; a.n = t->n; a.x = dx; a.x_rows = m; a.xs = ds; a.y16 = d16; a.y32 = d32;
    bool ok = to_device(dx, x, xb, s) && to_device(ds, x_scale, (size_t)m * 4, s) && cuda_ok(launch_i8_gemm(t, a, s), "i8 gemm launch");
    if (ok && y16) ok = to_host(y16, d16, yb * 2, s);
    if (ok && y32) ok = to_host(y32, d32, yb * 4, s);
    return ok && i8_status(t, s) == 0 ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

int omega_gpu_i8_status(const OmegaGpuI8Tensor *t, void *stream) {
    if (!t) return OMEGA_GPU_FP8_BAD_ARGS;
    Lock l;
    return i8_status(t, (cudaStream_t)stream);
}

int omega_gpu_i8_gemm_grouped_async(const OmegaGpuI8Tensor *t, uint32_t experts, uint32_t tile_rows, uint32_t max_tiles, uint64_t tiles_va, uint64_t header_va,
                                    uint64_t xmap_va, uint64_t ymap_va, uint64_t x_va, uint32_t x_rows, uint64_t x_scale_va, uint64_t y_bf16_va, uint64_t y_f32_va, void *stream) {
    if (!t || !experts || t->n % experts || !tile_rows || tile_rows > 256 || !max_tiles || !tiles_va || !header_va || !x_va || !x_rows || !x_scale_va || (!y_bf16_va && !y_f32_va)) return OMEGA_GPU_FP8_BAD_ARGS;
    if (max_tiles > I8_MAX_ROWS || x_rows > I8_MAX_ROWS) return OMEGA_GPU_FP8_TOO_LARGE;
    if ((uint64_t)max_tiles * ((t->n / experts + 127u) / 128u) > 0x7fffffffull) { set_error("i8 grouped: %u tiles of %u channels are more than 2^31 - 1 blocks of 128", max_tiles, t->n / experts); return OMEGA_GPU_FP8_TOO_LARGE; }
    if (((tiles_va | x_va | y_bf16_va | y_f32_va) & 15u) || ((header_va | xmap_va | ymap_va | x_scale_va) & 3u)) return OMEGA_GPU_FP8_BAD_ARGS;
    const int ready = async_ready();
    if (ready != OMEGA_GPU_FP8_OK) return ready;
    I8Launch a = {};
    a.m = max_tiles; a.n = t->n / experts; a.x = (const int8_t *)(uintptr_t)x_va; a.x_rows = x_rows; a.xs = (const float *)(uintptr_t)x_scale_va;
    a.y16 = (uint16_t *)(uintptr_t)y_bf16_va; a.y32 = (float *)(uintptr_t)y_f32_va; a.tiles = (const void *)(uintptr_t)tiles_va; a.header = (const uint32_t *)(uintptr_t)header_va;
    a.xmap = (const uint32_t *)(uintptr_t)xmap_va; a.ymap = (const uint32_t *)(uintptr_t)ymap_va; a.tile_rows = tile_rows;
    return cuda_ok(launch_i8_gemm(t, a, (cudaStream_t)stream), "i8 grouped launch") ? OMEGA_GPU_FP8_OK : OMEGA_GPU_FP8_CHIP_FAIL;
}

}  // extern "C"
