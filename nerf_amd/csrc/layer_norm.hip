// Layer norm over the last dimension and its backward pass, for the layers of networks the fused kernels do not cover:
//   mu = mean(x), s2 = mean((x - mu)^2), r = 1 / sqrt(s2 + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w, dx = r (g - mean(g) - xh mean(g xh)), dw = sum over rows of dy xh, db = sum over rows of dy
// All sums in fp32.  The mean is kept as a pair: mu1, the rounded sum over C, and mu2, the mean of x - mu1 -- the second pass
// over the row sums the differences for the variance anyway, and with mu2 a row whose offset is large against its spread loses
// nothing (a mean rounded to fp32 alone shifts every xh by up to 2^-24 |mu| / sigma).
#include <algorithm>
#include <type_traits>
#include "common.hpp"
#include "elem.hpp"
#include "wave_ops.hpp"

using namespace nerfhip;

namespace {

constexpr int LN_THREADS = 256;
constexpr int LN_SLICES = 1024;         // the most slices of the rows in the weight gradients' sums
constexpr int64_t LN_HELD = 16384;      // rows up to this length are held in registers
constexpr int LN_GROUPS = 2048;         // the most workgroups of the forward pass (us at 1024 / 2048 / 8192: 65536 x 256 fp32 24.4 / 22.2 / 22.0,
                                        // 16384 x 1024 bf16 13.7 / 13.2 / 14.8, 8192 x 8192 bf16 44.4 / 45.4 / 55.3)

template <typename T, int VEC>
__device__ __forceinline__ Loose<T, VEC> read_raw(const T* row, int i, int c) {      // zeros behind c
    if (i + VEC <= c) return *reinterpret_cast<const Loose<T, VEC>*>(row + i);
    Loose<T, VEC> v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v.e[e] = i + e < c ? row[i + e] : (T)0.0f;
    return v;
}
template <typename T, int VEC>
__device__ __forceinline__ void read_row(const T* row, int i, int c, float (&out)[VEC]) {
    const Loose<T, VEC> v = read_raw<T, VEC>(row, i, c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = (float)v.e[e];
}
template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* row, int i, int c, const float (&in)[VEC]) {
    if (i + VEC <= c) {
        Loose<T, VEC> v;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v.e[e] = (T)in[e];
        *reinterpret_cast<Loose<T, VEC>*>(row + i) = v;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (i + e < c) row[i + e] = (T)in[e];
    }
}

// a norm's weight or bias: fp32 or the rows' type, or absent
template <typename T>
struct Param {
    const void* p;
    int f32;
    __device__ __forceinline__ float at(int64_t i, float absent) const {
        return !p ? absent : f32 ? ((const float*)p)[i] : (float)((const T*)p)[i];
    }
    template <int VEC>
    __device__ __forceinline__ void read(int i, int c, float absent, float (&out)[VEC]) const {      // zeros behind c
        if (!p) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = i + e < c ? absent : 0.0f;
        } else if (f32) {
            read_row<float, VEC>((const float*)p, i, c, out);
        } else {
            read_row<T, VEC>((const T*)p, i, c, out);
        }
    }
};

template <int CTRL>
__device__ __forceinline__ float add_from(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// How a row is held: L lanes of WPR waves, VEC neighbouring elements at a time, CH times.
template <int L_, int WPR_, int VEC_, int CH_>
struct Shape {
    static constexpr int L = L_, WPR = WPR_, VEC = VEC_, CH = CH_;
    static constexpr int THREADS = WPR > 1 ? 64 * WPR : 256;
    static constexpr int PER_ROW = L * WPR;                  // threads of a row
    static constexpr int ROWS = THREADS / PER_ROW;           // rows a workgroup holds at once: one, or one or more for each wave
    static_assert(WPR == 1 || ROWS == 1);
    static constexpr int MAX_C = PER_ROW * VEC * CH;
    static constexpr int N = VEC * CH;
};

// the sum over a row's threads of K values, in every one of them; `part` holds K * WPR floats, another one for each call of an iteration
template <typename S, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* part) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (S::L == 16) {
            // (pairs that exchange: both lanes add the same two values, so that all sixteen end with the same bits; a mean that differed
            // from lane to lane would not be the one that the second pass corrects)
            v[k] = add_from<0xB1>(v[k]);       // quad_perm 1 0 3 2
            v[k] = add_from<0x4E>(v[k]);       // quad_perm 2 3 0 1
            v[k] = add_from<0x141>(v[k]);      // row_half_mirror
            v[k] = add_from<0x140>(v[k]);      // row_mirror
        } else {
            v[k] = wave_sum_f32(v[k]);
        }
    }
    if constexpr (S::WPR > 1) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) part[k * S::WPR + (threadIdx.x >> 6)] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = part[k * S::WPR];
#pragma unroll
            for (int w = 1; w < S::WPR; ++w) t += part[k * S::WPR + w];
            v[k] = t;
        }
    }
}

// One pass over memory: a row is read once, held in registers for both passes of the statistics, and written once.  A workgroup stays
// for many rows: the weight and the bias are read once, and the next row is under way while this one is worked on.  Bounded by memory:
// 65536 x 256 fp32 in 22 us (6.0 TB/s; 29 us with cold caches), 8192 x 4096 bf16 in 24 us (5.6 TB/s; 29), 10007 x 1537 fp16 in 18 us (3.4 TB/s:
// a quarter of the lanes is behind the row's end, and a row is short for what a workgroup's two sums cost).
template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS) k_ln_fwd_held(int64_t n, int c, const T* __restrict__ x, int64_t ldx, Param<T> w, Param<T> b, float eps,
                                                            T* __restrict__ y, int64_t ldy, float* __restrict__ stats) {
    __shared__ float part[2][2 * S::WPR];
    const int lane = threadIdx.x % S::PER_ROW, slot = threadIdx.x / S::PER_ROW;
    const float fc = (float)c;
    Loose<T, S::VEC> next[S::CH];
    auto request = [&](int64_t row) {
        const T* xr = x + (row < n ? row : n - 1) * ldx;
#pragma unroll
        for (int k = 0; k < S::CH; ++k) next[k] = read_raw<T, S::VEC>(xr, (k * S::PER_ROW + lane) * S::VEC, c);
    };
    request((int64_t)blockIdx.x * S::ROWS + slot);
    float wv[S::CH][S::VEC], bv[S::CH][S::VEC];
#pragma unroll
    for (int k = 0; k < S::CH; ++k) {
        const int i = (k * S::PER_ROW + lane) * S::VEC;
        w.read(i, c, 1.0f, wv[k]);
        b.read(i, c, 0.0f, bv[k]);
    }
    for (int64_t row0 = (int64_t)blockIdx.x * S::ROWS; row0 < n; row0 += (int64_t)gridDim.x * S::ROWS) {
        const int64_t row = row0 + slot;
        float v[S::CH][S::VEC], s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < S::CH; ++k)
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                v[k][e] = (float)next[k].e[e];
                s[0] += v[k][e];
            }
        if (row0 + (int64_t)gridDim.x * S::ROWS < n) request(row + (int64_t)gridDim.x * S::ROWS);
        row_sum<S, 1>(s, part[0]);
        const float mu1 = s[0] / fc;
        float d[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < S::CH; ++k) {
            const int i = (k * S::PER_ROW + lane) * S::VEC;
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                v[k][e] = i + e < c ? v[k][e] - mu1 : 0.0f;
                d[0] += v[k][e];
                d[1] += v[k][e] * v[k][e];
            }
        }
        row_sum<S, 2>(d, part[1]);
        const float mu2 = d[0] / fc, var = fmaxf(d[1] / fc - mu2 * mu2, 0.0f);
        const float r = (d[1] != d[1]) ? d[1] : 1.0f / sqrtf(var + eps);      // (fmaxf drops a NaN)
        if (row >= n) continue;
#pragma unroll
        for (int k = 0; k < S::CH; ++k) {
            const int i = (k * S::PER_ROW + lane) * S::VEC;
            if (i >= c) continue;
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) v[k][e] = (v[k][e] - mu2) * r * wv[k][e] + bv[k][e];
            write_row<T, S::VEC>(y + row * ldy, i, c, v[k]);
        }
        if (stats && lane == 0) {
            stats[row] = mu1;
            stats[n + row] = mu2;
            stats[2 * n + row] = r;
        }
    }
}

// x and dy are read once: dx is written and the weight's and bias's sums of this workgroup's rows stay in registers; they are left as
// partial[workgroup][0 | 1][column].  Bounded by memory: 65536 x 256 fp32 in 35 us (5.7 TB/s), 8192 x 4096 bf16 in 42 us (4.8 TB/s).
template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS, S::WPR > 4 ? 4 : 1) k_ln_bwd_held(int64_t n, int c, const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                            int64_t lddy, Param<T> w, const float* __restrict__ stats, T* __restrict__ dx,
                                                            int64_t lddx, float* __restrict__ partial) {
    __shared__ float part[2][2 * S::WPR];
    const int lane = threadIdx.x % S::PER_ROW, slot = threadIdx.x / S::PER_ROW;
    const float fc = (float)c;
    float wv[S::CH][S::VEC], sw[S::CH][S::VEC], sb[S::CH][S::VEC];
#pragma unroll
    for (int k = 0; k < S::CH; ++k) {
        w.read((k * S::PER_ROW + lane) * S::VEC, c, 1.0f, wv[k]);
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) sw[k][e] = sb[k][e] = 0.0f;
    }
    // (the next row is under way while this one is worked on, where a thread's registers allow it)
    constexpr bool AHEAD = S::WPR <= 4;
    Loose<T, S::VEC> nx[S::CH], ng[S::CH];
    auto request = [&](int64_t row) {
        const int64_t at = row < n ? row : n - 1;
#pragma unroll
        for (int k = 0; k < S::CH; ++k) {
            const int i = (k * S::PER_ROW + lane) * S::VEC;
            nx[k] = read_raw<T, S::VEC>(x + at * ldx, i, c);
            ng[k] = read_raw<T, S::VEC>(dy + at * lddy, i, c);
        }
    };
    if (AHEAD) request((int64_t)blockIdx.x * S::ROWS + slot);
    int odd = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * S::ROWS; row0 < n; row0 += (int64_t)gridDim.x * S::ROWS, odd ^= 1) {
        const int64_t row = row0 + slot;
        const bool live = row < n;
        const int64_t at = live ? row : n - 1;
        if (!AHEAD) request(row);
        const float mu1 = stats[at], mu2 = stats[n + at], r = stats[2 * n + at];
        float xh[S::CH][S::VEC], g[S::CH][S::VEC], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < S::CH; ++k)
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                xh[k][e] = (float)nx[k].e[e];
                g[k][e] = (float)ng[k].e[e];
            }
        if (AHEAD && row0 + (int64_t)gridDim.x * S::ROWS < n) request(row + (int64_t)gridDim.x * S::ROWS);
#pragma unroll
        for (int k = 0; k < S::CH; ++k) {
            const int i = (k * S::PER_ROW + lane) * S::VEC;
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                xh[k][e] = i + e < c ? (xh[k][e] - mu1 - mu2) * r : 0.0f;
                if (live) {
                    sw[k][e] += g[k][e] * xh[k][e];
                    sb[k][e] += g[k][e];
                }
                g[k][e] *= wv[k][e];
                s[0] += g[k][e];
                s[1] += g[k][e] * xh[k][e];
            }
        }
        if (!dx) continue;
        row_sum<S, 2>(s, part[odd]);
        const float ma = s[0] / fc, mq = s[1] / fc;
        if (live) {
#pragma unroll
            for (int k = 0; k < S::CH; ++k) {
                const int i = (k * S::PER_ROW + lane) * S::VEC;
                if (i >= c) continue;
                float o[S::VEC];
#pragma unroll
                for (int e = 0; e < S::VEC; ++e) o[e] = r * (g[k][e] - ma - xh[k][e] * mq);
                write_row<T, S::VEC>(dx + row * lddx, i, c, o);
            }
        }
    }
    if (!partial) return;
    // the workgroup's rows' sums together, in their order
    float* out = partial + (int64_t)blockIdx.x * 2 * c;
    if constexpr (S::ROWS > 1) {
        __shared__ float all[S::ROWS][S::MAX_C];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < S::CH; ++k)
#pragma unroll
                for (int e = 0; e < S::VEC; ++e) all[slot][(k * S::PER_ROW + lane) * S::VEC + e] = which ? sb[k][e] : sw[k][e];
            __syncthreads();
            for (int i = threadIdx.x; i < c; i += S::THREADS) {
                float t = all[0][i];
#pragma unroll
                for (int q = 1; q < S::ROWS; ++q) t += all[q][i];
                out[(int64_t)which * c + i] = t;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < S::CH; ++k) {
            const int i = (k * S::PER_ROW + lane) * S::VEC;
            if (i >= c) continue;
            write_row<float, S::VEC>(out, i, c, sw[k]);
            write_row<float, S::VEC>(out + c, i, c, sb[k]);
        }
    }
}

// ---- rows too long for registers: read again for every pass
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

template <typename T>
__global__ void __launch_bounds__(LN_THREADS) k_ln_fwd(int64_t n, int c, const T* __restrict__ x, int64_t ldx, Param<T> w,
                                                       Param<T> b, float eps, T* __restrict__ y, int64_t ldy,
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
        d2 = block_sum(d2, part);
        const float var = fmaxf(d2 / (float)c - mu2 * mu2, 0.0f);
        const float r = (d2 != d2) ? d2 : 1.0f / sqrtf(var + eps);      // (fmaxf drops a NaN)
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            float v = ((float)xr[i] - mu1 - mu2) * r;
            v = v * w.at(i, 1.0f) + b.at(i, 0.0f);
            y[row * ldy + i] = (T)v;
        }
        if (stats && threadIdx.x == 0) {
            stats[row] = mu1;
            stats[n + row] = mu2;
            stats[2 * n + row] = r;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LN_THREADS) k_ln_dx(int64_t n, int c, const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                      int64_t lddy, Param<T> w, const float* __restrict__ stats,
                                                      T* __restrict__ dx, int64_t lddx) {
    __shared__ float part[LN_THREADS / 64];
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const float mu1 = stats[row], mu2 = stats[n + row], r = stats[2 * n + row];
        const T *xr = x + row * ldx, *gr = dy + row * lddy;
        float a = 0.0f, q = 0.0f;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            const float g = (float)gr[i] * w.at(i, 1.0f);
            a += g;
            q += g * (((float)xr[i] - mu1 - mu2) * r);
        }
        const float ma = block_sum(a, part) / (float)c, mq = block_sum(q, part) / (float)c;
        for (int i = threadIdx.x; i < c; i += LN_THREADS) {
            const float g = (float)gr[i] * w.at(i, 1.0f);
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

// the slices' sums of 32 columns (of dw's C, then db's), in fp64, 32 slices at a time: 4 us for 1024 slices of 256 columns, 5 us for 768 of 4096
constexpr int LF_COLS = 32, LF_ROWS = 32;
template <typename W>
__global__ void __launch_bounds__(LF_COLS * LF_ROWS) k_ln_finish(int slices, int c, const float* __restrict__ partial, W* __restrict__ dw,
                                                                 W* __restrict__ db) {
    __shared__ double red[LF_ROWS][LF_COLS + 1];
    const int lane = threadIdx.x % LF_COLS, row = threadIdx.x / LF_COLS;
    const int64_t col = (int64_t)blockIdx.x * LF_COLS + lane;
    double s = 0.0;
    if (col < 2 * (int64_t)c) {
#pragma unroll 8
        for (int z = row; z < slices; z += LF_ROWS) s += (double)partial[(int64_t)z * 2 * c + col];
    }
    red[row][lane] = s;
    __syncthreads();
    if (row > 0 || col >= 2 * (int64_t)c) return;
#pragma unroll
    for (int k = 1; k < LF_ROWS; ++k) s += red[k][lane];
    if (col < c) {
        if (dw) dw[col] = (W)(float)s;
    } else if (db) {
        db[col - c] = (W)(float)s;
    }
}

// The shape that holds rows of c elements of `size` bytes: the fewest lanes at first (short rows: several to a wave, 16 bytes a lane), then
// more elements a lane, then more waves: 16 elements a lane of x, dy, the weight, both sums and the next row are what leaves four waves
// to a SIMD.  us forward / backward, taken and next best:
//   262144 x 64 fp32           4 elements of 16 lanes 22 / 35       8 elements 28 / 39
//   131072 x 128 bf16          8 elements of 16 lanes 14.5 / 22.6   2 elements of 64 lanes 34 / 35
//   65536 x 256 bf16           16 elements of 16 lanes 12.6 / 24    4 elements of 64 lanes 20.7 / 26.5
//   65536 x 256 fp32           4 elements of 64 lanes 22.4 / 35.9   16 elements of 16 lanes 21.7 / 35.7, but 1024 rows 3.0 / 6.3 against 2.5 / 5.4
//   32768 x 512 bf16           8 elements of 64 lanes 15.7 / 24     16 elements 19 / 34
//   16384 x 1024 bf16          one wave 13.6 / 23.4                 two waves 17 / 40
//   16384 x 1100 bf16          two waves 24 forward, four 43 backward   four waves 32, two 49
//   8192 x 4096 bf16           four waves 24 / 41                   eight waves 28 / 43
//   4096 x 8192 bf16           eight waves 26 / 49                  sixteen waves 29 / 46
//   2048 x 16384 bf16          sixteen waves 37 / 45                read again for each pass 82 / 129
template <bool FORWARD, int SIZE, typename F>
int with_shape(int64_t c, F&& f) {
    if (c <= 64) return f(Shape<16, 1, 4, 1>{});
    if (c <= 128) return f(Shape<16, 1, 8, 1>{});
    if (c <= 256) return f(std::conditional_t<SIZE == 2, Shape<16, 1, 8, 2>, Shape<64, 1, 4, 1>>{});
    if (c <= 512) return f(Shape<64, 1, 8, 1>{});
    if (c <= 1024) return f(Shape<64, 1, 8, 2>{});
    if (c <= 2048) return f(std::conditional_t<FORWARD, Shape<64, 2, 8, 2>, Shape<64, 4, 8, 1>>{});
    if (c <= 4096) return f(Shape<64, 4, 8, 2>{});
    if (c <= 8192) return f(Shape<64, 8, 8, 2>{});
    return f(Shape<64, 16, 8, 2>{});
}

// workgroups of the backward pass, each of which leaves one slice of the weight's gradient: enough to fill the machine, few enough
// that the slices (8 bytes a column each) stay a small part of the rows' own traffic and do not wait for one another.  (us at 256 / 512 /
// 768 / 1024 of them: 65536 x 256 fp32 53 / 36.5 / 35.5 / 35.5, 16384 x 1024 bf16 27 / 23 / 23.5 / 25.6, 16384 x 2048 bf16 72 / 44 / 40 / 39,
// 8192 x 4096 bf16 51 / 43 / 42 / 46, 8192 x 8192 bf16 98 / 94 / 110 / 110, 4096 x 16384 fp32 164 / 181 / 192 / 207)
template <int SIZE>
int slices_of(int64_t n, int64_t c) {
    if (n < 1) return 1;
    const int rows = c > LN_HELD ? 1 : with_shape<false, SIZE>(c, [](auto s) { return decltype(s)::ROWS; });
    const int64_t groups = (n + rows - 1) / rows;
    const int64_t most = c <= 512 || (c > 1024 && c <= 2048) ? LN_SLICES : c > 2048 && c <= 4096 ? LN_SLICES * 3 / 4 : c <= 8192 ? LN_SLICES / 2 : LN_SLICES / 4;
    // (few rows: a slice for each compute unit, more of them once four groups of rows share one: 2000 x 2000 bf16 17.2 -> 15.5 us, 4096 x 256 fp32
    // 8.2 -> 7.3, 300 x 8192 bf16 19 -> 16.5)
    return (int)std::min({groups, most, std::max(groups / 4, (int64_t)256)});
}

template <typename T>
int fwd(int64_t n, int c, const void* x, int64_t ldx, int w_f32, const void* w, const void* b, float eps, void* y, int64_t ldy, float* stats,
        hipStream_t stream) {
    const Param<T> wp{w, w_f32}, bp{b, w_f32};
    if (c > LN_HELD) {
        hipLaunchKernelGGL((k_ln_fwd<T>), dim3((unsigned)(n < 65536 ? n : 65536)), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx, wp, bp, eps,
                           (T*)y, ldy, stats);
        return launched("nerf_layer_norm_fwd");
    }
    return with_shape<true, sizeof(T)>(c, [&](auto shape) {
        using S = decltype(shape);
        const int64_t groups = (n + S::ROWS - 1) / S::ROWS;
        hipLaunchKernelGGL((k_ln_fwd_held<T, S>), dim3((unsigned)(groups < LN_GROUPS ? groups : LN_GROUPS)), dim3(S::THREADS), 0, stream, n, c, (const T*)x,
                           ldx, wp, bp, eps, (T*)y, ldy, stats);
        return launched("nerf_layer_norm_fwd");
    });
}

template <typename T>
int bwd(int64_t n, int c, const void* x, int64_t ldx, const void* dy, int64_t lddy, int w_f32, const void* w, const float* stats, void* dx,
        int64_t lddx, void* dw, void* db, float* ws, hipStream_t stream) {
    const Param<T> wp{w, w_f32};
    const int slices = slices_of<sizeof(T)>(n, c);
    float* part = dw || db ? ws : nullptr;
    if (!dx && !part) return 0;
    int rc = 0;
    if (c > LN_HELD || n == 0) {
        const unsigned cols = (unsigned)((c + LN_THREADS - 1) / LN_THREADS);
        if (dx && n > 0) {
            hipLaunchKernelGGL((k_ln_dx<T>), dim3((unsigned)(n < 65536 ? n : 65536)), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx,
                               (const T*)dy, lddy, wp, stats, (T*)dx, lddx);
            rc = launched("nerf_layer_norm_bwd");
            if (rc) return rc;
        }
        if (part) {
            hipLaunchKernelGGL((k_ln_dw<T>), dim3(cols, slices), dim3(LN_THREADS), 0, stream, n, c, (const T*)x, ldx, (const T*)dy, lddy, stats,
                               (n + slices - 1) / slices, part);
            rc = launched("nerf_layer_norm_bwd (partial sums)");
        }
    } else {
        rc = with_shape<false, sizeof(T)>(c, [&](auto shape) {
            using S = decltype(shape);
            hipLaunchKernelGGL((k_ln_bwd_held<T, S>), dim3((unsigned)slices), dim3(S::THREADS), 0, stream, n, c, (const T*)x, ldx, (const T*)dy,
                               lddy, wp, stats, (T*)dx, lddx, part);
            return launched("nerf_layer_norm_bwd");
        });
    }
    if (rc || !part) return rc;
    const dim3 grid((unsigned)((2 * (int64_t)c + LF_COLS - 1) / LF_COLS));
    if (w_f32) hipLaunchKernelGGL((k_ln_finish<float>), grid, dim3(LF_COLS * LF_ROWS), 0, stream, slices, c, part, (float*)dw, (float*)db);
    else hipLaunchKernelGGL((k_ln_finish<T>), grid, dim3(LF_COLS * LF_ROWS), 0, stream, slices, c, part, (T*)dw, (T*)db);
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
#define GO(T) return fwd<T>(n, (int)c, x, ldx, w_type == NERF_F32, w, b, (float)eps, y, ldy, stats, stream)
    if (type == NERF_F32) GO(float);
    if (type == NERF_BF16) GO(bf16_t);
    GO(f16_t);
#undef GO
}

int64_t nerf_layer_norm_workspace_floats(int64_t n, int64_t c) { return c < 1 ? 0 : (int64_t)std::max(slices_of<2>(n, c), slices_of<4>(n, c)) * 2 * c; }

int nerf_layer_norm_bwd(int64_t n, int64_t c, int type, const void* x, int64_t ldx, const void* dy, int64_t lddy, int w_type,
                        const void* w, const float* stats, void* dx, int64_t lddx, void* dw, void* db, float* workspace, void* stream_) {
    NERF_REQUIRE(n >= 0 && c >= 1 && c <= NERF_LAYER_NORM_MAX_C, "nerf_layer_norm_bwd: n=%lld c=%lld", (long long)n, (long long)c);
    NERF_REQUIRE(elem_type_ok(type) && (w_type == type || w_type == NERF_F32), "nerf_layer_norm_bwd: type=%d w_type=%d", type, w_type);
    NERF_REQUIRE(n <= 1 || (ldx >= c && lddy >= c && (!dx || lddx >= c)), "nerf_layer_norm_bwd: a row stride is less than c=%lld", (long long)c);
    NERF_REQUIRE(n == 0 || (x && dy && stats), "nerf_layer_norm_bwd: null pointer");
    NERF_REQUIRE(!(dw || db) || workspace, "nerf_layer_norm_bwd: null workspace");
    hipStream_t stream = as_stream(stream_);
#define GO(T) return bwd<T>(n, (int)c, x, ldx, dy, lddy, w_type == NERF_F32, w, stats, dx, lddx, dw, db, workspace, stream)
    if (type == NERF_F32) GO(float);
    if (type == NERF_BF16) GO(bf16_t);
    GO(f16_t);
#undef GO
}

}  // extern "C"
