// Products of matrices held in 8 bits (e4m3) with one power-of-two scale per row and 128 values of k:
//   C[i][j] = sum over blocks kb of 2^(ea[i][kb] + eb[j][kb]) sum over k in kb of a[i][k] b[j][k]   (+ bias[j], ReLU)
// and the quantisation that makes the operands.  A scale is the smallest power of two that takes its block's largest value to at
// most 448: x 2^-e is exact, so every value is rounded once, and applying it (E8M0 bytes, e + 127) rounds nothing.
//
// Which instruction multiplies: the codes are decoded to bf16 with their scale (4 bits into 8, the exponent range is fp32's: exact for
// values of magnitude from 2^-126 to below 2^128; smaller ones count as 0, larger ones as infinite) and multiplied by the bf16
// instruction, whose sums are within 2e-7 of the result (rms, k = 4096 and 65536).  Only the tiles of a bf16 output use the 8-bit
// instruction itself, which is twice as fast: it cuts the products of every eight consecutive k to multiples of 2^(E - 13), E the
// exponent of the largest of them, before it sums them in fp32, so that a result may lose up to 7 * 2^-13 of sum |a b|.  Error
// of 256 x 256 sums of 4096 and 65536 products, rms against the result's: 1.5e-5 on normally distributed operands, 5e-5 and 7.5e-5
// where the sizes of both vary along k by factors of exp(0.5 N) and exp(N), exp(N) and exp(2 N), always without a bias beyond 2e-6; the
// rounding to bf16 is 1.65e-3, which that raises by at most 0.1 %.  An fp16 output shows it (2.073e-4 -> 2.203e-4 in the worst of them),
// and so does an fp32 one.  A bf16 result that cancels to less than a hundredth of its products shows it too: whoever
// needs that takes an fp32 output.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "common.hpp"
#include "elem.hpp"
#include "wave_ops.hpp"

using namespace nerfhip;

namespace {

constexpr int KB = 128;       // values of k that share a scale

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

inline int64_t blocks_of(int64_t k) { return (k + KB - 1) / KB; }
inline int64_t code_stride(int64_t k) { return blocks_of(k) * KB; }
inline int64_t scale_stride(int64_t k) { return (blocks_of(k) + 3) / 4 * 4; }

// ---- quantisation ---------------------------------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ unsigned max_ror(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
    return o > v ? o : v;
}
__device__ __forceinline__ unsigned row16_max(unsigned v) {
    v = max_ror<0x121>(v);      // row_ror:1, 2, 4, 8 inside 16 lanes
    v = max_ror<0x122>(v);
    v = max_ror<0x124>(v);
    return max_ror<0x128>(v);
}

__device__ __forceinline__ unsigned mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr unsigned INF_BITS = 0x7f800000u;

// smallest e >= -126 with amax <= 448 * 2^e, from amax's bits (448 = 1.75 * 2^8)
__device__ __forceinline__ int scale_exp(unsigned amax) {
    const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }      // -126 <= e <= 127
// x * inv in e4m3, four to a word
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d, float inv) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
}
// What is not finite has no part in its block's largest value and becomes NaN.  A wave that meets such values (seen from its largest bits)
// takes them out, as zeros, remembers where they were, and puts the NaNs into the codes; the other waves pay for nothing.
template <int R>
__device__ __forceinline__ unsigned take_out(float (&v)[R][8]) {      // bit 8 q + e
    unsigned where = 0;
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool bad = mag_bits(v[q][e]) >= INF_BITS;
            where |= (bad ? 1u : 0u) << (8 * q + e);
            v[q][e] = bad ? 0.0f : v[q][e];
        }
    return where;
}
__device__ __forceinline__ unsigned nan_bytes(unsigned where, int first, int step) {      // NaN codes of four of the places
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (where >> (first + i * step) & 1u) * (0x7fu << (8 * i));
    return w;
}
__device__ __forceinline__ unsigned largest(const float (&v)[8]) {
    unsigned am = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) { const unsigned u = mag_bits(v[e]); am = u > am ? u : am; }
    return am;
}

constexpr int QT = 128;       // a workgroup quantises a tile of 128 x 128
constexpr int QLD = QT + 16;
constexpr int QR = 4, Q_THREADS = QT / QR * (QT / 8), Q_WAVES = Q_THREADS / 64;      // a thread's rows, of eight columns

// eight columns' values over a wave's four threads of each, to red[wave]
template <typename Op>
__device__ __forceinline__ void over_rows(unsigned (&v)[8], unsigned (*red)[QT], Op op) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = op(v[j], (unsigned)__shfl_xor((int)v[j], 16));
        v[j] = op(v[j], (unsigned)__shfl_xor((int)v[j], 32));
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) red[wave][lane * 8 + j] = v[j];
    }
}

// Along the columns alone: sixteen lanes hold a block of 128, a workgroup sixteen blocks that follow one another in memory.  Bounded by
// memory: 16384 x 4096 bf16 in 34 us, 5.9 TB/s.  (Four blocks a lane were slower at every size: 39 us there, 4 x 8192 3.6 us against 2.0.)
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_rows(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx,
                                                       unsigned blocks, uint8_t* __restrict__ codes, int64_t ldc, uint8_t* __restrict__ scales,
                                                       int64_t lds) {
    const int l = threadIdx.x & 15;
    const unsigned id = blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t row = id / blocks;
    const unsigned kb = id - (unsigned)row * blocks;
    if (row >= rows) return;
    const int64_t c = (int64_t)kb * KB + l * 8;
    float v[1][8];
    if (c + 8 <= cols) {
        load_vec<T, 8>(x + row * ldx + c, v[0]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[0][e] = c + e < cols ? (float)x[row * ldx + c + e] : 0.0f;
    }
    unsigned am = largest(v[0]), where = 0;
    if (__any(am >= INF_BITS)) {
        where = take_out(v);
        am = largest(v[0]);
    }
    const int ex = scale_exp(row16_max(am));
    const float inv = pow2(-ex);
    *reinterpret_cast<uint2*>(codes + row * ldc + c) = make_uint2(pack4(v[0][0], v[0][1], v[0][2], v[0][3], inv) | nan_bytes(where, 0, 1),
                                                                  pack4(v[0][4], v[0][5], v[0][6], v[0][7], inv) | nan_bytes(where, 4, 1));
    if (l == 0) {
        scales[row * lds + kb] = (uint8_t)(ex + 127);
        if (kb + 1 == blocks)
            for (int64_t z = blocks; z < lds; ++z) scales[row * lds + z] = 0;
    }
}

// codes / scales: along the columns (rows keep their order); codes_t / scales_t: of the transpose, along the rows; colsum: sums of the
// tile's columns, [tile row][cols].  mask: values whose mask entry is <= 0 count as 0 (the gradient of a ReLU's output).
// One pass over x whatever is asked for; the transposed codes are packed along the rows in registers and cross the workgroup as bytes.
// Bounded by memory where there is enough of it: both codes of 16384 x 4096 bf16 in 49 us, 5.5 TB/s; of 1001 x 333 in 9 us, most of it
// one pass through the instructions.  (Eight rows a thread: 70 us and 14 us; with every value looked at for being finite 61 us.)
template <typename T, bool ROWS>
__global__ void __launch_bounds__(Q_THREADS, 4) k_quantize(int64_t rows, int64_t cols, unsigned col_tiles, const T* __restrict__ x, int64_t ldx,
                                                  const T* __restrict__ mask, int64_t ldm, uint8_t* __restrict__ codes, int64_t ldc,
                                                  uint8_t* __restrict__ scales, int64_t lds, uint8_t* __restrict__ codes_t, int64_t ldct,
                                                  uint8_t* __restrict__ scales_t, int64_t ldst, float* __restrict__ colsum) {
    const unsigned row_tile = blockIdx.x / col_tiles, col_tile = blockIdx.x - row_tile * col_tiles, row_tiles = gridDim.x / col_tiles;
    const int64_t r0 = (int64_t)row_tile * QT, c0 = (int64_t)col_tile * QT;
    const int tid = threadIdx.x, rl = (tid >> 4) * QR, cl = (tid & 15) * 8;
    const int64_t c = c0 + cl;
    float v[QR][8];
    const bool inside = r0 + QT <= rows && c0 + QT <= cols;      // the whole tile
    const int nr = (int)(rows - r0 - rl < QR ? rows - r0 - rl : QR), nc = (int)(cols - c < 8 ? cols - c : 8);      // this thread's valid part, possibly < 1
    const T* src = x + (r0 + rl) * ldx + c;
    if (inside) {
#pragma unroll
        for (int q = 0; q < QR; ++q) load_vec<T, 8>(src + q * ldx, v[q]);
    } else {
#pragma unroll
        for (int q = 0; q < QR; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[q][e] = (q < nr && e < nc) ? (float)src[q * ldx + e] : 0.0f;
    }
    if (mask) {
        const T* gate = mask + (r0 + rl) * ldm + c;
#pragma unroll
        for (int q = 0; q < QR; ++q) {
            float m[8];
            if (inside) {
                load_vec<T, 8>(gate + q * ldm, m);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) m[e] = (q < nr && e < nc) ? (float)gate[q * ldm + e] : 1.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[q][e] = m[e] <= 0.0f ? 0.0f : v[q][e];
        }
    }
    // the columns: sums and largest values of the waves' rows, then one thread for each column
    __shared__ unsigned red[2][Q_WAVES][QT];
    __shared__ __attribute__((aligned(16))) float unit[QT];      // 2^-e of the columns
    if (colsum) {
        unsigned sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float t = v[0][j];
#pragma unroll
            for (int q = 1; q < QR; ++q) t += v[q][j];
            sum[j] = __float_as_uint(t);
        }
        over_rows(sum, red[0], [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); });
    }
    unsigned row_am[QR], where = 0, top = 0;
#pragma unroll
    for (int q = 0; q < QR; ++q) {
        row_am[q] = largest(v[q]);
        top = row_am[q] > top ? row_am[q] : top;
    }
    const bool some_bad = __any(top >= INF_BITS);
    if (some_bad) {
        where = take_out(v);
#pragma unroll
        for (int q = 0; q < QR; ++q) row_am[q] = largest(v[q]);
    }
    if (ROWS) {
#pragma unroll
        for (int q = 0; q < QR; ++q) {
            const int64_t r = r0 + rl + q;
            const int ex = scale_exp(row16_max(row_am[q]));
            const float inv = pow2(-ex);
            if (r < rows) {
                uint2 w = make_uint2(pack4(v[q][0], v[q][1], v[q][2], v[q][3], inv), pack4(v[q][4], v[q][5], v[q][6], v[q][7], inv));
                if (some_bad) {
                    w.x |= nan_bytes(where, 8 * q, 1);
                    w.y |= nan_bytes(where, 8 * q + 4, 1);
                }
                *reinterpret_cast<uint2*>(codes + r * ldc + c) = w;
                if ((tid & 15) == 0) {
                    scales[r * lds + col_tile] = (uint8_t)(ex + 127);
                    if (col_tile + 1 == col_tiles)
                        for (int64_t z = col_tiles; z < lds; ++z) scales[r * lds + z] = 0;
                }
            }
        }
    }
    if (codes_t) {
        unsigned am[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            am[j] = 0;
#pragma unroll
            for (int q = 0; q < QR; ++q) { const unsigned u = mag_bits(v[q][j]); am[j] = u > am[j] ? u : am[j]; }
        }
        over_rows(am, red[1], [](unsigned a, unsigned b) { return a > b ? a : b; });
    }
    __syncthreads();
    if (tid < QT) {
        const int64_t col = c0 + tid;
        if (colsum && col < cols) {
            float t = __uint_as_float(red[0][0][tid]);
#pragma unroll
            for (int w = 1; w < Q_WAVES; ++w) t += __uint_as_float(red[0][w][tid]);
            colsum[(int64_t)row_tile * cols + col] = t;
        }
        if (codes_t) {
            unsigned am = red[1][0][tid];
#pragma unroll
            for (int w = 1; w < Q_WAVES; ++w) am = red[1][w][tid] > am ? red[1][w][tid] : am;
            const int ex = scale_exp(am);
            unit[tid] = pow2(-ex);
            if (col < cols) {
                scales_t[col * ldst + row_tile] = (uint8_t)(ex + 127);
                if (row_tile + 1 == row_tiles)
                    for (int64_t z = row_tiles; z < ldst; ++z) scales_t[col * ldst + z] = 0;
            }
        }
    }
    if (!codes_t) return;
    __shared__ __attribute__((aligned(16))) uint8_t bytes[QT * QLD];      // [column][row]
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float inv = unit[cl + j];
        unsigned w = pack4(v[0][j], v[1][j], v[2][j], v[3][j], inv);
        if (some_bad) w |= nan_bytes(where, j, 8);
        // (sixteen bytes of a column lie at their place ^ (column / 16): the lanes of a wave write to all banks)
        *reinterpret_cast<unsigned*>(bytes + (cl + j) * QLD + (rl ^ ((cl >> 4) << 4))) = w;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < QT * QT / 16 / Q_THREADS; ++q) {
        const int piece = tid + Q_THREADS * q, col = piece >> 3, k = (piece & 7) * 16;
        if (c0 + col < cols) *reinterpret_cast<uint4*>(codes_t + (c0 + col) * ldct + r0 + k) = *reinterpret_cast<const uint4*>(bytes + col * QLD + (k ^ ((col >> 4) << 4)));
    }
}

// the tiles' sums of 64 columns, in fp64, sixteen tiles at a time (512 tiles of 256 columns: 4.6 us)
constexpr int CF_ROWS = 16;
template <typename T>
__global__ void __launch_bounds__(64 * CF_ROWS) k_colsum_finish(int64_t tiles, int64_t cols, const float* __restrict__ part, T* __restrict__ out) {
    __shared__ double red[CF_ROWS][64];
    const int lane = threadIdx.x & 63, row = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 4
        for (int64_t t = row; t < tiles; t += CF_ROWS) s += (double)part[t * cols + c];
    }
    red[row][lane] = s;
    __syncthreads();
    if (row == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < CF_ROWS; ++k) s += red[k][lane];
        out[c] = (T)(float)s;
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------------
struct Product {
    const uint8_t *a, *b, *sa, *sb;
    int64_t m, n;
    int64_t ldk, lds;         // row strides of codes and scales
    int blocks;               // 128-blocks of k
    const void* bias;
    int bias_f32, relu;
    void* c;
    int64_t ldc;
};

template <typename T>
__device__ __forceinline__ float finish(float v, const Product& p, int64_t col) {
    if (p.bias) v += p.bias_f32 ? ((const float*)p.bias)[col] : (float)((const T*)p.bias)[col];
    if (p.relu) v = v > 0.0f ? v : (v != v ? v : 0.0f);      // keeps a NaN
    return v;
}

// a lane's 32 of the 128 bytes of a block: the 16 at 16 g and the 16 at 64 + 16 g (any division of k will do that both operands share;
// with this one an instruction reads 64 bytes of a row together)
__device__ __forceinline__ i32x8 load32(const uint8_t* p) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(p), y = *reinterpret_cast<const i32x4*>(p + 64);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ bf16x8 decode8(int lo, int hi, float scale) {
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
// acc += a b^T over one block of k: a lane holds 32 of the 128 values of row (lane & 15) of either operand, and that row's scale byte
__device__ __forceinline__ f32x4 mul_decoded(i32x8 a, int sa, i32x8 b, int sb, f32x4 acc) {
    const float fa = __uint_as_float((unsigned)sa << 23), fb = __uint_as_float((unsigned)sb << 23);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decode8(a[2 * q], a[2 * q + 1], fa), decode8(b[2 * q], b[2 * q + 1], fb), acc, 0, 0, 0);
    return acc;
}

// Few rows: a workgroup owns 16 columns of C and up to 16 MT rows; each of its waves takes an eighth of the blocks of k, straight from
// memory into the instruction's registers, four blocks requested at a time, and the waves add up through LDS.  The weight's codes
// are read once: that is what bounds it (4 x 8192 x 8192 in 13.9-14.3 us, 4.7-4.9 TB/s).
constexpr int FEW_WAVES = 8, FEW_U = 4;
template <typename T, int MT>
__global__ void __launch_bounds__(64 * FEW_WAVES) k_product_few(Product p) {
    __shared__ f32x4 red[FEW_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t j0 = (int64_t)blockIdx.x * 16, i0 = (int64_t)blockIdx.y * 16 * MT;
    const int64_t jb = j0 + r < p.n ? j0 + r : p.n - 1;
    const uint8_t *bp = p.b + jb * p.ldk + 16 * g, *sbp = p.sb + jb * p.lds;
    const uint8_t *ap[MT], *sap[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t ia = i0 + 16 * t + r < p.m ? i0 + 16 * t + r : p.m - 1;
        ap[t] = p.a + ia * p.ldk + 16 * g;
        sap[t] = p.sa + ia * p.lds;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0, 0, 0, 0};
    // (a wave's blocks in fours, whose scales are one word of a row)
    const int fours = (p.blocks + 3) / 4, per = (fours + FEW_WAVES - 1) / FEW_WAVES;
    const int q1 = (wave + 1) * per < fours ? (wave + 1) * per : fours;
    for (int q = wave * per; q < q1; ++q) {
        const int kb = 4 * q;
        i32x8 b[FEW_U];
#pragma unroll
        for (int u = 0; u < FEW_U; ++u) b[u] = load32(bp + (int64_t)(kb + u < p.blocks ? kb + u : p.blocks - 1) * KB);
        const unsigned sb = *reinterpret_cast<const unsigned*>(sbp + kb);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const unsigned sa = *reinterpret_cast<const unsigned*>(sap[t] + kb);
            i32x8 a[FEW_U];
#pragma unroll
            for (int u = 0; u < FEW_U; ++u) a[u] = load32(ap[t] + (int64_t)(kb + u < p.blocks ? kb + u : p.blocks - 1) * KB);
#pragma unroll
            for (int u = 0; u < FEW_U; ++u) {
                if (kb + u >= p.blocks) break;
                const int ea = (int)(sa >> 8 * u & 255u), eb = (int)(sb >> 8 * u & 255u);
                acc[t] = mul_decoded(a[u], ea, b[u], eb, acc[t]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += FEW_WAVES) {
        f32x4 s = red[0][t][lane];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) s += red[w][t][lane];
        const int64_t col = j0 + r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t row = i0 + 16 * t + 4 * g + e;
            if (row < p.m && col < p.n) ((T*)p.c)[row * p.ldc + col] = (T)finish<T>(s[e], p, col);
        }
    }
}

// ---- tiles --------------------------------------------------------------------------------------------------------------------
// A workgroup of four waves owns a BM x BN tile of C, a wave a quarter of it in 32 x 32 pieces.  Per block of k, (BM + BN) rows of 128
// bytes go from memory straight into LDS (global_load_lds, 16 bytes a lane), into one of two images.  A block is multiplied in two
// halves of 64: while the first multiplies out of registers, the second's fragments are read, after which the image is done with;
// from then on the rows of the block after the next are asked for in its place, one request beside each matrix instruction, and
// while the second half multiplies, the first fragments of the next block are read.  So a request has a block of multiplication to
// arrive and a read a quarter of one.  (The requests take half of the address path's time: all in one half block they held the matrix
// instructions up, 8192^3 in 440 us against 416.)  The 16-byte pieces of a row are stored in the order piece ^ (row / 2 & 7): the
// sixteen lanes whose 16-byte reads the LDS serves together hold rows that differ in this and the row's parity, so they cover all 64
// banks (piece ^ (row & 7) cost as many cycles again in conflicts).
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mul32_fp8(i32x8 a, int sa, i32x8 b, int sb, f32x16 acc) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 0, 0, 0, sa, 0, sb);
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }      // in a scalar register

template <int ROWS>
struct Stage {      // one operand's rows on their way into LDS
    static constexpr int N = ROWS / 32;      // instructions of a wave per block, eight rows each
    const uint8_t* base;
    unsigned offset[N];      // of this lane's 16 bytes; rows behind the last stand for the last
    __device__ __forceinline__ void aim(const uint8_t* p, int64_t row0, int64_t rows, int64_t ldk) {
        base = p + row0 * ldk;
        const int lane = threadIdx.x & 63, wave = wave_id();
        const int last = (int)(rows - row0 < ROWS ? rows - row0 : ROWS) - 1;
        const int r = lane >> 3;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = 8 * (wave + 4 * i) + r;
            offset[i] = (unsigned)(row < last ? row : last) * (unsigned)ldk + (((lane & 7) ^ (row >> 1 & 7)) << 4);
        }
    }
    __device__ __forceinline__ void issue(int i, int kb, uint8_t* image) const {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + (int64_t)kb * KB + offset[i]),
                                         (__attribute__((address_space(3))) void*)(image + 8 * (wave_id() + 4 * i) * KB), 16, 0, 0);
    }
};

// where a lane's 32 of the 64 bytes of either half of row `row` lie in an image: pieces 4 h + 2 g and the one behind it
struct Piece {
    int x[2], y[2];
    __device__ __forceinline__ Piece(int row, int g) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[h] = row * KB + (((4 * h + 2 * g) ^ (row >> 1 & 7)) << 4);
            y[h] = row * KB + (((4 * h + 2 * g + 1) ^ (row >> 1 & 7)) << 4);
        }
    }
    __device__ __forceinline__ i32x8 read(const uint8_t* image, int h, int t) const {      // of the row 32 t further (the order of its pieces is the same)
        const i32x4 p = *reinterpret_cast<const i32x4*>(image + x[h] + 32 * t * KB), q = *reinterpret_cast<const i32x4*>(image + y[h] + 32 * t * KB);
        return __builtin_shufflevector(p, q, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// eight rows x COLS columns of a wave's LDS band to out[row][col], each lane 16 bytes of a row at a time
template <typename T, int COLS, int LD>
struct Out {
    static constexpr int VEC = 16 / sizeof(T), GROUPS = COLS / VEC, ROWS = 64 / GROUPS;
    static_assert(8 % ROWS == 0);
    T* out;
    const float* from;
    int64_t m, ldo;
    int rl, cols;      // cols of this lane's VEC are in the matrix
    float floor, bias[VEC];
    __device__ __forceinline__ Out(const float* band, const Product& p, int64_t col0, T* o, int64_t ld, bool last) : m(p.m), ldo(ld) {
        const int lane = threadIdx.x & 63, c = (lane % GROUPS) * VEC;
        const int64_t col = col0 + c;
        rl = lane / GROUPS;
        from = band + rl * LD + c;
        out = o + col;
        cols = col + VEC <= p.n ? VEC : (col < p.n ? (int)(p.n - col) : 0);
        floor = last && p.relu ? 0.0f : -INFINITY;
#pragma unroll
        for (int e = 0; e < VEC; ++e) bias[e] = 0.0f;
        auto take = [&](const auto* b) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) bias[e] = (float)b[col + e < p.n ? col + e : p.n - 1];
        };
        if (last && p.bias) {
            if (p.bias_f32) take((const float*)p.bias);
            else take((const T*)p.bias);
        }
    }
    // WHOLE: the wave's rows and columns are all in the matrix
    template <bool WHOLE>
    __device__ __forceinline__ void rows(int64_t row0) const {
        constexpr int R = 8 / ROWS;
        float v[R][VEC];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(from + i * ROWS * LD + e);
#pragma unroll
                for (int d = 0; d < 4; ++d) v[i][e + d] = q[d];
            }
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] += bias[e];
                v[i][e] = v[i][e] < floor ? 0.0f : v[i][e];      // keeps a NaN
            }
            const int64_t row = row0 + i * ROWS + rl;
            T* dst = out + row * ldo;
            if (WHOLE) {
                store_vec<T, VEC>(dst, v[i]);
            } else if (row < m) {
                if (cols == VEC) {
                    store_vec<T, VEC>(dst, v[i]);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (e < cols) dst[e] = (T)v[i][e];
                }
            }
        }
    }
};

template <typename T, int BM, int BN>
struct TileLds {      // two images, two sets of scale words, a band of eight rows for each wave on its way out
    static constexpr int IMAGE = (BM + BN) * KB, WORDS = (BM + BN) * 4, LD = BN / 2 + 4, BAND = 8 * LD * 4;
    static constexpr int WORDS_AT = 2 * IMAGE, BAND_AT = WORDS_AT + 2 * WORDS, BYTES = BAND_AT + 4 * BAND;
};

// A workgroup stays for several tiles, and k runs on from one into the next: the requests for a tile's first blocks go out while the
// one before it is still multiplied and written.  (A workgroup for each tile spent 11.5 us of 103 on the way out and in; bf16 of
// 8192^3: 413 -> 390 us.)  Scales come once in four blocks: a word of a row costs the cache a lookup like a whole line, and with every
// block they were half of them (8192 x 8192 x 16384: 848 -> 746 us).
// 256 x 256, bf16 of random codes: 8192^3 in 385-418 us over the boards (2.6-2.9 PFLOP/s), 16384 x 8192 x 4096 in 409-441 us; of zeros 277 us -- the board's power
// limit takes the rest, the matrix pipe is busy 81 % of the cycles, 15 % are waits at the two barriers of a block.  128 x 128, fp32 and fp16:
// 8192^3 in 845 us (1.30 PFLOP/s, of the bf16 instruction), 16384 x 8192 x 4096 in 917-934 us, 65536 x 256 x 256 in 18-20 us (4.2-4.7 TB/s).
template <typename T, int BM, int BN>
__global__ void __launch_bounds__(256) k_product_tile(Product p, int tiles_m, int tiles_n, int blocks_per_slice, float* __restrict__ partial) {
    constexpr bool DECODED = !std::is_same_v<T, bf16_t>;      // which instruction: see the top of this file
    constexpr int MT = BM / 64, NT = BN / 64;      // 32 x 32 pieces of a wave
    constexpr int M = MT * NT, P = MT + NT;        // P <= M: a piece beside each of the first P
    static_assert(P <= M);
    constexpr bool LONG = M >= 16;                 // half a block takes long enough for barriers of its own
    using Lds = TileLds<T, BM, BN>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 31, g = lane >> 5;
    const int total = tiles_m * tiles_n;
    const int kb0 = blockIdx.z * blocks_per_slice;
    const int kb1 = kb0 + blocks_per_slice < p.blocks ? kb0 + blocks_per_slice : p.blocks;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);

    // neighbouring tiles on one XCD (workgroups go to the eight XCDs in turn), in bands of four rows of tiles
    auto corner = [&](int id, int64_t& i0, int64_t& j0) {
        constexpr int BAND = 4;
        const int per = total / 8, extra = total % 8, x = id & 7;
        id = x * per + (x < extra ? x : extra) + (id >> 3);
        const int band = id / (BAND * tiles_n), in_band = id - band * BAND * tiles_n;
        const int band_rows = tiles_m - band * BAND < BAND ? tiles_m - band * BAND : BAND;
        i0 = (int64_t)(band * BAND + in_band % band_rows) * BM;
        j0 = (int64_t)(in_band / band_rows) * BN;
    };

    // requests: the rows of one operand each, and the scales, four blocks' a word per row, which come along with every block
    constexpr int SROWS = (BM + BN) / 4, WORD_ISSUES = SROWS / 64;      // rows of a wave
    Stage<BM> sa;
    Stage<BN> sb;
    const uint8_t* srow[WORD_ISSUES];
    auto aim = [&](int64_t i0, int64_t j0) {
        sa.aim(p.a, i0, p.m, p.ldk);
        sb.aim(p.b, j0, p.n, p.ldk);
#pragma unroll
        for (int i = 0; i < WORD_ISSUES; ++i) {
            const int row = SROWS * wave + 64 * i + lane;      // A's rows, then B's
            if (SROWS * wave + 64 * i < BM) srow[i] = p.sa + (i0 + row < p.m ? i0 + row : p.m - 1) * p.lds;
            else srow[i] = p.sb + (j0 + row - BM < p.n ? j0 + row - BM : p.n - 1) * p.lds;
        }
    };
    constexpr int NA = Stage<BM>::N, N = NA + Stage<BN>::N;      // this wave's row instructions of a block
    auto issue = [&](int i, int kb, int place) {
        uint8_t* image = lds + place * Lds::IMAGE;
        if (i < NA) sa.issue(i, kb, image);
        else sb.issue(i - NA, kb, image + BM * KB);
    };
    auto issue_words = [&](int kb, int place) {
#pragma unroll
        for (int i = 0; i < WORD_ISSUES; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(srow[i] + 4 * (int64_t)(kb >> 2)),
                                             (__attribute__((address_space(3))) void*)(lds + Lds::WORDS_AT + place * Lds::WORDS + (SROWS * wave + 64 * i) * 4), 4, 0, 0);
    };

    // reads
    const Piece pa(wm + r, g), pb(wn + r, g);
    i32x8 a0[MT], b0[NT], a1[MT], b1[NT];
    unsigned wa[MT], wb[NT], na[MT], nb[NT];
    auto fetch = [&](int i, int place, int h, i32x8 (&a)[MT], i32x8 (&b)[NT]) {      // piece i of a half block's MT + NT
        const uint8_t* image = lds + place * Lds::IMAGE;
        if (i < MT) a[i] = pa.read(image, h, i);
        else b[i - MT] = pb.read(image + BM * KB, h, i - MT);
    };
    auto fetch_words = [&](int place) {
        const unsigned* w = reinterpret_cast<const unsigned*>(lds + Lds::WORDS_AT + place * Lds::WORDS);
#pragma unroll
        for (int t = 0; t < MT; ++t) na[t] = w[wm + 32 * t + r];
#pragma unroll
        for (int u = 0; u < NT; ++u) nb[u] = w[BM + wn + 32 * u + r];
    };

    f32x16 acc[MT][NT];
    auto clear = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][u][e] = 0.0f;
    };
    // One half block multiplies out of a, b; between its instructions and in this order `beside(i)` places reads and requests.  (One wave
    // per SIMD: what is not placed between matrix instructions, which take 64 cycles each, is waited for.)
    auto multiply = [&](const i32x8 (&a)[MT], const i32x8 (&b)[NT], auto beside) {
        if constexpr (!DECODED) {
#pragma unroll
            for (int i = 0; i < M; ++i) {
                acc[i / NT][i % NT] = mul32_fp8(a[i / NT], (int)wa[i / NT], b[i % NT], (int)wb[i % NT], acc[i / NT][i % NT]);
                beside(i);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < M; ++i) beside(i);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                bf16x8 ad[MT], bd[NT];
#pragma unroll
                for (int t = 0; t < MT; ++t) ad[t] = decode8(a[t][2 * q], a[t][2 * q + 1], __uint_as_float((wa[t] & 255u) << 23));
#pragma unroll
                for (int u = 0; u < NT; ++u) bd[u] = decode8(b[u][2 * q], b[u][2 * q + 1], __uint_as_float((wb[u] & 255u) << 23));
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int u = 0; u < NT; ++u) acc[t][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ad[t], bd[u], acc[t][u], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto scales_of = [&](int kb) {
        const int sh = 8 * (kb & 3);
#pragma unroll
        for (int t = 0; t < MT; ++t) wa[t] = na[t] >> sh;
#pragma unroll
        for (int u = 0; u < NT; ++u) wb[u] = nb[u] >> sh;
    };
    // out through LDS, eight rows of the wave's columns at a time, so that a store is 16 bytes of a row (or fp32 partial sums likewise)
    float* const band = reinterpret_cast<float*>(lds + Lds::BAND_AT) + wave * 8 * Lds::LD;
    auto write_by = [&](const auto& out, int64_t i0, auto whole) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) band[(e + 4 * g) * Lds::LD + 32 * u + r] = acc[t][u][4 * q + e];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // (one wave's LDS instructions run in order)
                out.template rows<decltype(whole)::value>(i0 + wm + 32 * t + 8 * q);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
    };
    auto write = [&](int64_t i0, int64_t j0) {
        if (!LONG && partial) {
            write_by(Out<float, 32 * NT, Lds::LD>(band, p, j0 + wn, partial + (int64_t)blockIdx.z * p.m * p.n, p.n, false), i0, std::false_type{});
        } else {
            const Out<T, 32 * NT, Lds::LD> out(band, p, j0 + wn, (T*)p.c, p.ldc, true);
            if (i0 + BM <= p.m && j0 + BN <= p.n) write_by(out, i0, std::true_type{});
            else write_by(out, i0, std::false_type{});
        }
    };

    int64_t i0, j0;
    corner(blockIdx.x, i0, j0);
    aim(i0, j0);
    clear();
    if constexpr (LONG) {
        constexpr int X = P + 1, Y = 3, EARLY = M - X;
        // The block asked for runs two ahead of the one multiplied: a tile's last two blocks (kb1 >= 2) ask for the next tile's first
        // two.  Behind the last tile its own first rows come once more, for nobody.  Blocks use the two images in turn, and words of four
        // blocks' scales the two sets.
        int image = 0, words = 0;      // words: the set of the tile's first word
        // block ask_kb is asked for, its scales into the set ask_set; the next block's scales are in next_set, moved by next_shift
        auto step = [&](int ask_kb, int ask_set, int next_set, int next_shift) {
            multiply(a0, b0, [&](int i) {
                if (i < P) fetch(i, image, 1, a1, b1);
                if (i == X) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // everyone is done with this block's image
                if (i >= X) issue(i - X, ask_kb, image);
            });
            multiply(a1, b1, [&](int i) {
                if (EARLY + i < N) issue(EARLY + i, ask_kb, image);
                else if (EARLY + i == N && (ask_kb & 3) == 0) issue_words(ask_kb, ask_set);
                if (i == Y)      // the next block is in LDS: out are at most the requests made since
                    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(EARLY + Y + 1) : "memory");
                if (i > Y && i - Y - 1 < P) fetch(i - Y - 1, image ^ 1, 0, a0, b0);
                if (i == Y + P + 1) fetch_words(next_set);
                if (i == M - 1) scales_of(next_shift);
            });
            image ^= 1;
        };
        issue_words(0, 0);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < N; ++i) issue(i, kb, kb);
        }
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
#pragma unroll
        for (int i = 0; i < P; ++i) fetch(i, 0, 0, a0, b0);
        fetch_words(0);
        scales_of(0);
        for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
            for (int kb = 0; kb < kb1 - 2; ++kb) step(kb + 2, words ^ ((kb + 2) >> 2 & 1), words ^ ((kb + 1) >> 2 & 1), kb + 1);
            const int next = tile + (int)gridDim.x < total ? tile + (int)gridDim.x : tile;
            const int next_words = words ^ ((kb1 + 3) >> 2 & 1);
            int64_t ni, nj;
            corner(next, ni, nj);
            aim(ni, nj);
#pragma unroll 1
            for (int q = 0; q < 2; ++q) step(q, next_words, q ? next_words : words ^ ((kb1 - 1) >> 2 & 1), q ? 0 : kb1 - 1);
            words = next_words;
            write(i0, j0);
            clear();
            i0 = ni;
            j0 = nj;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // nothing may arrive in LDS that is another workgroup's by then
    } else {
        auto place_of = [&](int kb) { return (kb >> 2) & 1; };
        auto block = [&](int kb, auto more) {      // more: there are two blocks behind this one
            scales_of(kb);
            multiply(a0, b0, [&](int i) { if (i < P) fetch(i, kb & 1, 1, a1, b1); });
            // this wave's rows of the next block are in LDS, then everyone's; and everyone is done with this one's image
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            multiply(a1, b1, [&](int i) {
                if constexpr (decltype(more)::value) {
                    if (i == 0 && ((kb + 2) & 3) == 0) issue_words(kb + 2, place_of(kb + 2));
#pragma unroll
                    for (int q = i * N / M; q < (i + 1) * N / M; ++q) issue(q, kb + 2, kb & 1);
                }
                if (i < P) fetch(i, (kb + 1) & 1, 0, a0, b0);
                if (i == M / 2) fetch_words(place_of(kb + 1));
            });
        };
        issue_words(kb0, place_of(kb0));
#pragma unroll
        for (int i = 0; i < N; ++i) issue(i, kb0, kb0 & 1);
        if (kb0 + 1 < kb1) {
            issue_words(kb0 + 1, place_of(kb0 + 1));
#pragma unroll
            for (int i = 0; i < N; ++i) issue(i, kb0 + 1, (kb0 + 1) & 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < P; ++i) fetch(i, kb0 & 1, 0, a0, b0);
        fetch_words(place_of(kb0));
        int kb = kb0;
        for (; kb + 2 < kb1; ++kb) block(kb, std::true_type{});
        for (; kb < kb1; ++kb) block(kb, std::false_type{});      // (behind the last block an image's old rows are read and not used)
        write(i0, j0);
    }
}

// c = act(sum over the slices of k + bias): four groups of 64 threads take a quarter of the slices each, in their order, and their sums
// are added in theirs; a thread holds four values that follow one another in the partial sums (64 slices of 256 x 256: 4.7 us)
template <typename T>
__global__ void __launch_bounds__(256) k_product_join(Product p, int slices, const float* __restrict__ partial) {
    __shared__ float4 red[3][64];
    const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
    const int64_t size = p.m * p.n, i = ((int64_t)blockIdx.x * 64 + lane) * 4;
    const int per = (slices + 3) / 4, z0 = group * per, z1 = z0 + per < slices ? z0 + per : slices;
    float4 s = make_float4(0, 0, 0, 0);
    if (i + 4 <= size && (size & 3) == 0) {
#pragma unroll 8
        for (int z = z0; z < z1; ++z) {
            const float4 q = *reinterpret_cast<const float4*>(partial + z * size + i);
            s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
        }
    } else {
        float t[4] = {0, 0, 0, 0};
        for (int z = z0; z < z1; ++z)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < size) t[e] += partial[z * size + i + e];
        s = make_float4(t[0], t[1], t[2], t[3]);
    }
    if (group > 0) red[group - 1][lane] = s;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        const float4 o = red[q][lane];
        s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i + e >= size) break;
        const int64_t row = (i + e) / p.n, col = i + e - row * p.n;
        ((T*)p.c)[row * p.ldc + col] = (T)finish<T>(v[e], p, col);
    }
}

// How a product is cut, from its sizes alone.
struct Plan {
    int tile;           // 0: few rows; else the tile's edge
    int slices;         // of k
    int blocks_per_slice;
};
// The machine's compute units, which cut a product and are the most workgroups that stay for several large tiles.  A constant and not the
// current device's count: workspaces are sized without a device, and the same product gives the same bits on every one (on a
// partition of the machine with fewer of them the workgroups take turns).
constexpr int UNITS = 256;
Plan plan_of(int64_t m, int64_t n, int64_t k, int type) {
    const int64_t blocks = blocks_of(k);
    // Few rows or tiles: what either takes in us, fitted to both at 4 to 64 rows and n x k from 256 x 256 to 8192 x 8192 and 1024 x 65536.
    // (8192 x 8192: 4 rows 13.9 / 17.4, 16 rows 18.6 / 18.1, 64 rows 42.8 / 20.9; 1024 x 1024, 64 rows: 5.5 / 8.9;
    // 1024 x 65536, 4 rows: 47 / 18, few workgroups with a long way each)
    const double few = 2.4 + (double)k * (n > 4096 ? n : 4096) * (17 + m) / 1.34e8, many = 7.5 + (double)n * k / 6.4e6;
    // And a k above 2^22 whatever m and n, with 64-bit offsets throughout, where a tile's rows are 32 bits apart (they would reach to 2^24;
    // 256 x 256 over 2^22 values of k by tiles 1.1 ms, over 2^22 + 300 by few rows 10.7 ms).
    if ((m <= 64 && few <= many) || k > (1 << 22)) return {0, 1, (int)blocks};
    auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
    const int64_t small = tiles(128);
    // Large tiles or small: large ones use the matrix instruction better, and a tile costs them more.  What either takes in us, fitted to
    // 2048 x 2048 to 5632 x 5632 at k = 4096 and 512 and to 65536 x 256 x 256; a round that is not full takes less than a full one.  (bf16,
    // large / small: 4096 x 4096 x 4096 62 / 74, 2560 x 3584 x 4096 45 / 55, 5632 x 5632 x 4096 105 / 135, 2048 x 2048 x 4096 61 / 26,
    // 4096 x 4096 x 512 19.5 / 17.2.)  Large tiles ask for blocks two ahead, so that they need two.
    const double r = (double)tiles(256) / UNITS, q = (double)small / (2 * UNITS);
    const double large_us = (r + 2 * std::ceil(r)) / 3 * (13.4 + 1.3 * blocks), small_us = (q + std::ceil(q)) / 2 * (4.5 + 1.02 * blocks);
    if (type == NERF_BF16 && blocks > 1 && large_us < small_us) return {256, 1, (int)blocks};
    // Few small tiles leave compute units idle: k is cut in slices, whose sums a second launch joins.  A block takes 0.76 us, the join
    // 5 us and what the partial sums cost to write and to read.  (256 x 256 x 65536 fp32: 1 slice 390, 16 slices 34.5, 64 slices 21.0;
    // 1024 x 1024 x 1024: 1 slice 7.3, 2 slices 12.6.)
    const int64_t most = small < UNITS ? std::min(UNITS / small, blocks) : 1;
    const double block_us = 0.76, sum_us = 2e-6 * (double)m * n;
    int64_t slices = std::min(std::max((int64_t)(std::sqrt(blocks * block_us / sum_us) + 0.5), (int64_t)1), most);
    if (blocks * block_us / slices + 5 + slices * sum_us >= blocks * block_us) slices = 1;
    const int64_t per = (blocks + slices - 1) / slices;
    return {128, (int)((blocks + per - 1) / per), (int)per};
}

template <typename T>
int product(const Product& p, int64_t k, int type, float* ws, hipStream_t stream) {
    const Plan plan = plan_of(p.m, p.n, k, type);
    if (plan.tile == 0) {
        const int mt = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
        const int64_t gx = (p.n + 15) / 16, gy = (p.m + 16 * mt - 1) / (16 * mt);
        if (gx > 0x7fffff || gy > 65535) return fail(NERF_E_ARG, "nerf_fp8_matmul: %lld x %lld is more than one launch covers", (long long)p.m, (long long)p.n);
#define GO(MT) hipLaunchKernelGGL((k_product_few<T, MT>), dim3((unsigned)gx, (unsigned)gy), dim3(64 * FEW_WAVES), 0, stream, p)
        if (mt == 1) GO(1); else if (mt == 2) GO(2); else GO(4);
#undef GO
        return launched("nerf_fp8_matmul");
    }
    const int64_t tm = (p.m + plan.tile - 1) / plan.tile, tn = (p.n + plan.tile - 1) / plan.tile;
    if (tm * tn > 0xffffff) return fail(NERF_E_ARG, "nerf_fp8_matmul: %lld x %lld is more than one launch covers", (long long)p.m, (long long)p.n);
    const int64_t wgs = plan.tile == 256 && tm * tn > UNITS ? UNITS : tm * tn;
    const dim3 grid((unsigned)wgs, 1, (unsigned)plan.slices);
    float* part = plan.slices > 1 ? ws : nullptr;
    if (plan.slices > 1 && !ws) return fail(NERF_E_ARG, "nerf_fp8_matmul: null workspace");
#define GO(E)                                                                                                                        \
    do {                                                                                                                             \
        constexpr size_t bytes = TileLds<T, E, E>::BYTES; \
        const hipError_t e = lds_limit_once((const void*)&k_product_tile<T, E, E>, bytes);                                           \
        if (e != hipSuccess) return fail(NERF_E_LAUNCH, "nerf_fp8_matmul: %s", hipGetErrorString(e));                                \
        hipLaunchKernelGGL((k_product_tile<T, E, E>), grid, dim3(256), bytes, stream, p, (int)tm, (int)tn, plan.blocks_per_slice, part); \
    } while (0)
    if constexpr (std::is_same_v<T, bf16_t>) {
        if (plan.tile == 256) GO(256); else GO(128);
    } else {
        GO(128);
    }
#undef GO
    const int rc = launched("nerf_fp8_matmul");
    if (rc || !part) return rc;
    hipLaunchKernelGGL((k_product_join<T>), dim3((unsigned)((p.m * p.n + 255) / 256)), dim3(256), 0, stream, p, plan.slices, part);
    return launched("nerf_fp8_matmul (join)");
}

template <typename T>
int quantize(int64_t rows, int64_t cols, const T* x, int64_t ldx, const T* mask, int64_t ldm, uint8_t* codes, uint8_t* scales,
             uint8_t* codes_t, uint8_t* scales_t, int sum_type, void* col_sum, float* ws, hipStream_t stream) {
    const int64_t ldc = code_stride(cols), lds = scale_stride(cols), ldct = code_stride(rows), ldst = scale_stride(rows);
    if (codes_t || col_sum || mask) {
        const int64_t col_tiles = (cols + QT - 1) / QT, tiles_all = (rows + QT - 1) / QT * col_tiles;
        if (tiles_all > 0xffffff) return fail(NERF_E_ARG, "nerf_fp8_quantize: %lld x %lld is more than one launch covers", (long long)rows, (long long)cols);
#define GO(R)                                                                                                                        \
    hipLaunchKernelGGL((k_quantize<T, R>), dim3((unsigned)tiles_all), dim3(Q_THREADS), 0, stream, rows, cols, (unsigned)col_tiles, x, ldx, mask, ldm, \
                       codes, ldc, scales, lds, codes_t, ldct, scales_t, ldst, col_sum ? ws : (float*)nullptr)
        if (codes) GO(true); else GO(false);
#undef GO
    } else {
        const int64_t blocks = blocks_of(cols), wgs = (rows * blocks + 15) / 16;
        if (wgs > 0xffffff) return fail(NERF_E_ARG, "nerf_fp8_quantize: %lld x %lld is more than one launch covers", (long long)rows, (long long)cols);
        hipLaunchKernelGGL((k_quantize_rows<T>), dim3((unsigned)wgs), dim3(256), 0, stream, rows, cols, x, ldx, (unsigned)blocks, codes, ldc, scales, lds);
    }
    const int rc = launched("nerf_fp8_quantize");
    if (rc || !col_sum) return rc;
    const dim3 cgrid((unsigned)((cols + 63) / 64));
    const int64_t tiles = (rows + QT - 1) / QT;
    if (sum_type == NERF_F32) hipLaunchKernelGGL((k_colsum_finish<float>), cgrid, dim3(64 * CF_ROWS), 0, stream, tiles, cols, ws, (float*)col_sum);
    else hipLaunchKernelGGL((k_colsum_finish<T>), cgrid, dim3(64 * CF_ROWS), 0, stream, tiles, cols, ws, (T*)col_sum);
    return launched("nerf_fp8_quantize (sums)");
}

}  // namespace

extern "C" {

int64_t nerf_fp8_code_stride(int64_t k) { return k < 1 ? 0 : code_stride(k); }
int64_t nerf_fp8_scale_stride(int64_t k) { return k < 1 ? 0 : scale_stride(k); }
int64_t nerf_fp8_quantize_workspace_floats(int64_t rows, int64_t cols) { return rows < 1 || cols < 1 ? 0 : (rows + QT - 1) / QT * cols; }

int nerf_fp8_quantize(int64_t rows, int64_t cols, int type, const void* x, int64_t ldx, const void* mask, int64_t ldm, uint8_t* codes,
                      uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, int sum_type, void* col_sum, float* workspace, void* stream_) {
    NERF_REQUIRE(!col_sum || sum_type == type || sum_type == NERF_F32, "nerf_fp8_quantize: type=%d sum_type=%d", type, sum_type);
    NERF_REQUIRE(rows >= 0 && cols >= 1, "nerf_fp8_quantize: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    NERF_REQUIRE(elem_type_ok(type), "nerf_fp8_quantize: type=%d", type);
    NERF_REQUIRE(rows <= (int64_t)QT * 0x7fffff && cols <= (int64_t)QT * 65535, "nerf_fp8_quantize: %lld x %lld is more than one launch covers",
                 (long long)rows, (long long)cols);      // (and the products of tiles below)
    NERF_REQUIRE(rows <= 1 || (ldx >= cols && (!mask || ldm >= cols)), "nerf_fp8_quantize: a row stride is less than cols=%lld", (long long)cols);
    if (rows == 0) return 0;
    NERF_REQUIRE(x && (!codes == !scales) && (!codes_t == !scales_t) && (codes || codes_t || col_sum) && (!col_sum || workspace),
                 "nerf_fp8_quantize: null pointer");
    NERF_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(codes_t)) & 15) == 0,
                 "nerf_fp8_quantize: codes start at a multiple of 16 bytes");
    hipStream_t stream = as_stream(stream_);
#define GO(T) return quantize<T>(rows, cols, (const T*)x, ldx, (const T*)mask, ldm, codes, scales, codes_t, scales_t, sum_type, col_sum, workspace, stream)
    if (type == NERF_F32) GO(float);
    if (type == NERF_BF16) GO(bf16_t);
    GO(f16_t);
#undef GO
}

int nerf_fp8_matmul(int64_t m, int64_t n, int64_t k, const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales,
                    int bias_type, const void* bias, int relu, int type, void* c, int64_t ldc, float* workspace, void* stream_) {
    NERF_REQUIRE(m >= 0 && n >= 0 && k >= 1 && k <= 0x7fffffff, "nerf_fp8_matmul: m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
    NERF_REQUIRE(elem_type_ok(type) && (!bias || bias_type == type || bias_type == NERF_F32), "nerf_fp8_matmul: type=%d bias_type=%d", type, bias_type);
    NERF_REQUIRE(m <= 1 || ldc >= n, "nerf_fp8_matmul: ldc=%lld is less than n=%lld", (long long)ldc, (long long)n);
    if (m == 0 || n == 0) return 0;
    NERF_REQUIRE(a && a_scales && b && b_scales && c, "nerf_fp8_matmul: null pointer");
    NERF_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0 &&
                 ((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) & 3) == 0,
                 "nerf_fp8_matmul: codes start at a multiple of 16 bytes, scales of 4");
    Product p{a, b, a_scales, b_scales, m, n, code_stride(k), scale_stride(k), (int)blocks_of(k), bias, bias_type == NERF_F32, relu, c, ldc};
    hipStream_t stream = as_stream(stream_);
    if (type == NERF_F32) return product<float>(p, k, type, workspace, stream);
    if (type == NERF_BF16) return product<bf16_t>(p, k, type, workspace, stream);
    return product<f16_t>(p, k, type, workspace, stream);
}

int nerf_fp8_matmul_tile(int64_t m, int64_t n, int64_t k, int type) { return m < 1 || n < 1 || k < 1 ? 0 : plan_of(m, n, k, type).tile; }

int64_t nerf_fp8_matmul_workspace_floats(int64_t m, int64_t n, int64_t k, int type) {
    if (m < 1 || n < 1 || k < 1) return 0;
    const Plan plan = plan_of(m, n, k, type);
    return plan.slices > 1 ? plan.slices * m * n : 0;
}

// What a layer keeps for its backward pass and needs for a while, as offsets of 256 bytes' multiples into two buffers.
namespace {
inline int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }
struct Held {      // a quantised matrix [rows, k] inside a buffer
    int64_t codes, scales, end;
    Held(int64_t at, int64_t rows, int64_t k) : codes(at), scales(at + up256(rows * code_stride(k))), end(scales + up256(rows * scale_stride(k))) {}
};
struct Kept {
    Held xt, wt;      // x^T [n_in, n], w^T [n_in, n_out]
    Kept(int64_t n, int64_t n_in, int64_t n_out, bool dx, bool dw) : xt(0, dw ? n_in : 0, n), wt(xt.end, dx ? n_in : 0, n_out) {}
};
struct Forward {
    Held x, w;
    int64_t part, end;
    Forward(int64_t n, int64_t n_in, int64_t n_out, int type)
        : x(0, n, n_in), w(x.end, n_out, n_in), part(w.end), end(part + up256(4 * nerf_fp8_matmul_workspace_floats(n, n_out, n_in, type))) {}
};
struct Backward {
    Held g, gt;       // dy [n, n_out], dy^T [n_out, n]
    int64_t sums, part, end;
    Backward(int64_t n, int64_t n_in, int64_t n_out, int type, int w_type)
        : g(0, n, n_out), gt(g.end, n_out, n), sums(gt.end), part(sums + up256(4 * nerf_fp8_quantize_workspace_floats(n, n_out))), end(part) {
        const int64_t a = nerf_fp8_matmul_workspace_floats(n, n_in, n_out, type), b = nerf_fp8_matmul_workspace_floats(n_out, n_in, n, w_type);
        end += up256(4 * (a > b ? a : b));      // (one product after the other)
    }
};
}  // namespace

int64_t nerf_linear_fp8_kept_bytes(int64_t n, int64_t n_in, int64_t n_out, int needs_dx, int needs_dw) {
    return n < 1 || n_in < 1 || n_out < 1 ? 0 : Kept(n, n_in, n_out, needs_dx != 0, needs_dw != 0).wt.end;
}
int64_t nerf_linear_fp8_workspace_bytes(int64_t n, int64_t n_in, int64_t n_out, int type, int w_type, int backward) {
    if (n < 1 || n_in < 1 || n_out < 1) return 0;
    return backward ? Backward(n, n_in, n_out, type, w_type).end : Forward(n, n_in, n_out, type).end;
}

int nerf_linear_fp8_fwd(int64_t n, int64_t n_in, int64_t n_out, int type, const void* x, int64_t ldx, int w_type, const void* w, int64_t ldw,
                        const uint8_t* w_codes, const uint8_t* w_scales, int bias_type, const void* bias, int relu, void* y, void* kept,
                        int needs_dx, int needs_dw, void* workspace, void* stream) {
    NERF_REQUIRE(n >= 0 && n_in >= 1 && n_out >= 1, "nerf_linear_fp8_fwd: n=%lld n_in=%lld n_out=%lld", (long long)n, (long long)n_in, (long long)n_out);
    NERF_REQUIRE(elem_type_ok(type) && (!w || w_type == type || w_type == NERF_F32), "nerf_linear_fp8_fwd: type=%d w_type=%d", type, w_type);
    if (n == 0) return 0;
    NERF_REQUIRE(x && y && workspace && (w || (w_codes && w_scales && !kept)), "nerf_linear_fp8_fwd: null pointer");
    NERF_REQUIRE(((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(kept)) & 255) == 0,
                 "nerf_linear_fp8_fwd: kept and workspace start at a multiple of 256 bytes");
    uint8_t* ws = (uint8_t*)workspace;
    uint8_t* keep = (uint8_t*)kept;
    const Forward f(n, n_in, n_out, type);
    const bool kx = keep && needs_dw, kw = keep && needs_dx;
    const Kept k(n, n_in, n_out, kw, kx);
    int rc = nerf_fp8_quantize(n, n_in, type, x, ldx, nullptr, 0, ws + f.x.codes, ws + f.x.scales, kx ? keep + k.xt.codes : nullptr,
                               kx ? keep + k.xt.scales : nullptr, NERF_F32, nullptr, nullptr, stream);
    if (rc) return rc;
    if (w) {
        rc = nerf_fp8_quantize(n_out, n_in, w_type, w, ldw, nullptr, 0, ws + f.w.codes, ws + f.w.scales, kw ? keep + k.wt.codes : nullptr,
                               kw ? keep + k.wt.scales : nullptr, NERF_F32, nullptr, nullptr, stream);
        if (rc) return rc;
        w_codes = ws + f.w.codes;
        w_scales = ws + f.w.scales;
    }
    return nerf_fp8_matmul(n, n_out, n_in, ws + f.x.codes, ws + f.x.scales, w_codes, w_scales, bias_type, bias, relu, type, y, n_out,
                           (float*)(ws + f.part), stream);
}

int nerf_linear_fp8_bwd(int64_t n, int64_t n_in, int64_t n_out, int type, const void* dy, int64_t lddy, const void* y, const void* kept,
                        int needs_dx, int needs_dw, void* dx, int w_type, void* dw, int bias_type, void* db, void* workspace, void* stream) {
    NERF_REQUIRE(n >= 1 && n_in >= 1 && n_out >= 1, "nerf_linear_fp8_bwd: n=%lld n_in=%lld n_out=%lld", (long long)n, (long long)n_in, (long long)n_out);
    NERF_REQUIRE(elem_type_ok(type) && (w_type == type || w_type == NERF_F32) && (!db || bias_type == type || bias_type == NERF_F32),
                 "nerf_linear_fp8_bwd: type=%d w_type=%d bias_type=%d", type, w_type, bias_type);
    if (!dx && !dw && !db) return 0;
    NERF_REQUIRE(dy && workspace && ((!dx && !dw) || kept), "nerf_linear_fp8_bwd: null pointer");
    NERF_REQUIRE((!dx || needs_dx) && (!dw || needs_dw), "nerf_linear_fp8_bwd: a gradient is asked for that the forward pass kept nothing for");
    NERF_REQUIRE(((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(kept)) & 255) == 0,
                 "nerf_linear_fp8_bwd: kept and workspace start at a multiple of 256 bytes");
    uint8_t* ws = (uint8_t*)workspace;
    const uint8_t* keep = (const uint8_t*)kept;
    const Backward b(n, n_in, n_out, type, w_type);
    const Kept k(n, n_in, n_out, needs_dx != 0, needs_dw != 0);
    int rc = nerf_fp8_quantize(n, n_out, type, dy, lddy, y, n_out, dx ? ws + b.g.codes : nullptr, dx ? ws + b.g.scales : nullptr,
                               dw ? ws + b.gt.codes : nullptr, dw ? ws + b.gt.scales : nullptr, bias_type, db, (float*)(ws + b.sums), stream);
    if (rc) return rc;
    if (dx) {
        rc = nerf_fp8_matmul(n, n_in, n_out, ws + b.g.codes, ws + b.g.scales, keep + k.wt.codes, keep + k.wt.scales, type, nullptr, 0, type, dx, n_in,
                             (float*)(ws + b.part), stream);
        if (rc) return rc;
    }
    if (!dw) return 0;
    return nerf_fp8_matmul(n_out, n_in, n, ws + b.gt.codes, ws + b.gt.scales, keep + k.xt.codes, keep + k.xt.scales, w_type, nullptr, 0, w_type, dw, n_in,
                           (float*)(ws + b.part), stream);
}

}  // extern "C"
