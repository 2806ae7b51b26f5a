// Layer norm over the last dimension and its backward pass, for the layers of networks the fused kernels do not cover:
//   mu = mean(x), s2 = mean((x - mu)^2), r = 1 / sqrt(s2 + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w, dx = r (g - mean(g) - xh mean(g xh)), dw = sum over rows of dy xh, db = sum over rows of dy
// All sums in fp32.  The mean is kept as a pair: mu1, the rounded sum over C, and mu2, the mean of x - mu1 -- the second pass
// over the row sums the differences for the variance anyway, and with mu2 a row whose offset is large against its spread loses
// nothing (a mean rounded to fp32 alone shifts every xh by up to 2^-24 |mu| / sigma).
#include "common.hpp"
#include "elem.hpp"
#include "wave_ops.hpp"

using namespace nerfhip;

namespace {

constexpr int LN_THREADS = 256;
constexpr int LN_SLICES = 256;      // slices of the rows in the weight gradients' sums

__device__ __forceinline__ float block_sum(float v, float* part) {
    v = wave_sum_f32(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < LN_THREADS / 64; ++w) t += part[w];
    return t;
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) k_ln_fwd(int64_t n, int c, const T* __restrict__ x, int64_t ldx, const W* __restrict__ w,
                                                       const W* __restrict__ b, float eps, T* __restrict__ y, int64_t ldy,
                                                       float* __restrict__ stats) {
    __shared__ float part[LN_THREADS / 64];
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const T* xr = x + row * ldx;
        float s = 0.0f;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) s += (float)xr[i];
        const float mu1 = block_sum(s, part) / (float)c;
        float d1 = 0.0f, d2 = 0.0f;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            const float d = (float)xr[i] - mu1;
            d1 += d;
            d2 += d * d;
        }
        const float mu2 = block_sum(d1, part) / (float)c;
        const float var = fmaxf(block_sum(d2, part) / (float)c - mu2 * mu2, 0.0f);
        const float r = 1.0f / sqrtf(var + eps);
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            float v = ((float)xr[i] - mu1 - mu2) * r;
            if (w) v *= (float)w[i];
            if (b) v += (float)b[i];
            y[row * ldy + i] = (T)v;
        }
        if (stats && threadIdx.x == 0) {
            stats[row] = mu1;
            stats[n + row] = mu2;
            stats[2 * n + row] = r;
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) k_ln_dx(int64_t n, int c, const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                      int64_t lddy, const W* __restrict__ w, const float* __restrict__ stats,
                                                      T* __restrict__ dx, int64_t lddx) {
    __shared__ float part[LN_THREADS / 64];
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const float mu1 = stats[row], mu2 = stats[n + row], r = stats[2 * n + row];
        const T *xr = x + row * ldx, *gr = dy + row * lddy;
        float a = 0.0f, q = 0.0f;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            const float g = (float)gr[i] * (w ? (float)w[i] : 1.0f);
            a += g;
            q += g * (((float)xr[i] - mu1 - mu2) * r);
        }
        const float ma = block_sum(a, part) / (float)c, mq = block_sum(q, part) / (float)c;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            const float g = (float)gr[i] * (w ? (float)w[i] : 1.0f);
            dx[row * lddx + i] = (T)(r * (g - ma - (((float)xr[i] - mu1 - mu2) * r) * mq));
        }
    }
}

// partial[slice][0][col] = sum over the slice's rows of dy xh, partial[slice][1][col] of dy
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) k_ln_dw(int64_t n, int c, const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                      int64_t lddy, const float* __restrict__ stats, int64_t rows_per_slice,
                                                      float* __restrict__ partial) {
    const int col = blockIdx.x * LN_THREADS + threadIdx.x;
    if (col >= c) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per_slice, r1 = r0 + rows_per_slice < n ? r0 + rows_per_slice : n;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t row = r0; row < r1; ++row) {
        const float g = (float)dy[row * lddy + col];
        sw += g * (((float)x[row * ldx + col] - stats[row] - stats[n + row]) * stats[2 * n + row]);
        sb += g;
    }
    partial[((int64_t)blockIdx.y * 2) * c + col] = sw;
    partial[((int64_t)blockIdx.y * 2 + 1) * c + col] = sb;
}

template <typename W>
__global__ void __launch_bounds__(LN_THREADS) k_ln_finish(int slices, int c, const float* __restrict__ partial, W* __restrict__ dw,
                                                          W* __restrict__ db) {
    const int col = blockIdx.x * LN_THREADS + threadIdx.x;
    if (col >= c) return;
    double sw = 0.0, sb = 0.0;
    for (int z = 0; z < slices; ++z) {
        sw += (double)partial[((int64_t)z * 2) * c + col];
        sb += (double)partial[((int64_t)z * 2 + 1) * c + col];
    }
    if (dw) dw[col] = (W)(float)sw;
    if (db) db[col] = (W)(float)sb;
}

int slices_of(int64_t n) { return (int)(n < LN_SLICES ? (n < 1 ? 1 : n) : LN_SLICES); }

template <typename T, typename W>
int fwd(int64_t n, int c, const void* x, int64_t ldx, const void* w, const void* b, float eps, void* y, int64_t ldy, float* stats,
        hipStream_t stream) {
    const unsigned grid = (unsigned)(n < 65536 ? n : 65536);
    hipLaunchKernelGGL((k_ln_fwd<T, W>), dim3(grid), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx, (const W*)w, (const W*)b, eps,
                       (T*)y, ldy, stats);
    return launched("nerf_layer_norm_fwd");
}

template <typename T, typename W>
int bwd(int64_t n, int c, const void* x, int64_t ldx, const void* dy, int64_t lddy, const void* w, const float* stats, void* dx,
        int64_t lddx, void* dw, void* db, float* ws, hipStream_t stream) {
    if (dx && n > 0) {
        const unsigned grid = (unsigned)(n < 65536 ? n : 65536);
        hipLaunchKernelGGL((k_ln_dx<T, W>), dim3(grid), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx, (const T*)dy, lddy,
                           (const W*)w, stats, (T*)dx, lddx);
        const int rc = launched("nerf_layer_norm_bwd");
        if (rc) return rc;
    }
    if (!dw && !db) return 0;
    const int slices = slices_of(n);
    const unsigned cols = (unsigned)((c + LN_THREADS - 1) / LN_THREADS);
    hipLaunchKernelGGL((k_ln_dw<T>), dim3(cols, slices), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx, (const T*)dy, lddy, stats,
                       (n + slices - 1) / slices, ws);
    const int rc = launched("nerf_layer_norm_bwd (partial sums)");
    if (rc) return rc;
    hipLaunchKernelGGL((k_ln_finish<W>), dim3(cols), dim3(LN_THREADS), 0, stream, slices, c, ws, (W*)dw, (W*)db);
    return launched("nerf_layer_norm_bwd (sums)");
}

}  // namespace

extern "C" {

int nerf_layer_norm_fwd(int64_t n, int64_t c, int type, const void* x, int64_t ldx, int w_type, const void* w, const void* b, double eps,
                        void* y, int64_t ldy, float* stats, void* stream_) {
    NERF_REQUIRE(n >= 0 && c >= 1 && c <= NERF_LAYER_NORM_MAX_C, "nerf_layer_norm_fwd: n=%lld c=%lld", (long long)n, (long long)c);
    NERF_REQUIRE(elem_type_ok(type) && (w_type == type || w_type == NERF_F32), "nerf_layer_norm_fwd: type=%d w_type=%d", type, w_type);
    NERF_REQUIRE(n <= 1 || (ldx >= c && ldy >= c), "nerf_layer_norm_fwd: ldx=%lld ldy=%lld are less than c=%lld", (long long)ldx,
                 (long long)ldy, (long long)c);
    NERF_REQUIRE(eps >= 0.0, "nerf_layer_norm_fwd: eps=%g", eps);
    if (n == 0) return 0;
    NERF_REQUIRE(x && y, "nerf_layer_norm_fwd: null pointer");
    hipStream_t stream = as_stream(stream_);
#define GO(T, W) return fwd<T, W>(n, (int)c, x, ldx, w, b, (float)eps, y, ldy, stats, stream)
    if (type == NERF_F32) GO(float, float);
    if (type == NERF_BF16) { if (w_type == NERF_F32) GO(bf16_t, float); GO(bf16_t, bf16_t); }
    if (w_type == NERF_F32) GO(f16_t, float);
    GO(f16_t, f16_t);
#undef GO
}

int64_t nerf_layer_norm_workspace_floats(int64_t n, int64_t c) { return (int64_t)slices_of(n) * 2 * (c < 0 ? 0 : c); }

int nerf_layer_norm_bwd(int64_t n, int64_t c, int type, const void* x, int64_t ldx, const void* dy, int64_t lddy, int w_type,
                        const void* w, const float* stats, void* dx, int64_t lddx, void* dw, void* db, float* workspace, void* stream_) {
    NERF_REQUIRE(n >= 0 && c >= 1 && c <= NERF_LAYER_NORM_MAX_C, "nerf_layer_norm_bwd: n=%lld c=%lld", (long long)n, (long long)c);
    NERF_REQUIRE(elem_type_ok(type) && (w_type == type || w_type == NERF_F32), "nerf_layer_norm_bwd: type=%d w_type=%d", type, w_type);
    NERF_REQUIRE(n <= 1 || (ldx >= c && lddy >= c && (!dx || lddx >= c)), "nerf_layer_norm_bwd: a row stride is less than c=%lld", (long long)c);
    NERF_REQUIRE(n == 0 || (x && dy && stats), "nerf_layer_norm_bwd: null pointer");
    NERF_REQUIRE(!(dw || db) || workspace, "nerf_layer_norm_bwd: null workspace");
    hipStream_t stream = as_stream(stream_);
#define GO(T, W) return bwd<T, W>(n, (int)c, x, ldx, dy, lddy, w, stats, dx, lddx, dw, db, workspace, stream)
    if (type == NERF_F32) GO(float, float);
    if (type == NERF_BF16) { if (w_type == NERF_F32) GO(bf16_t, float); GO(bf16_t, bf16_t); }
    if (w_type == NERF_F32) GO(f16_t, float);
    GO(f16_t, f16_t);
#undef GO
}

}  // extern "C"
