// AdamW over any number of tensors, wherever they lie, in one launch per NERF_ADAMW_BATCH of them (plus one small launch that
// counts the steps and forms the coefficients that depend on the count):
//   m += (1 - beta1)(g - m),  v += (1 - beta2)(g^2 - v),
//   p -= lr wd p + lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// in fp32 (the moments as increments, so that their fixed point does not depend on how beta rounds); 16-bit parameters are
// rounded from an fp32 master copy.
//
// States in 8 bits: per block of 128 consecutive elements of a tensor the scales sm = max |m| / 448 and sv = max v / 57344 (fp32, at
// least 1e-38 unless the block is 0), m / sm held in e4m3 and v / sv in e5m2.  Both are rounded stochastically: with beta2 = 0.999 a step moves v by at most a
// thousandth of what it lacks, far below half a step of any 8-bit format, so that rounded to nearest it would stand still; rounded up with
// the probability of the remainder its mean is kept.  The random bits are a hash of (element, step): the same run gives the
// same bits.  A positive v never becomes 0, because it divides.
//
// Bounded by memory: 235.8 M bf16 parameters with their master copies (30 bytes each) in 1.30 ms, 5.4 TB/s; 59.1 M fp32 with states in 8 bits
// (16.1 bytes) in 173-185 us, 5.1-5.5 TB/s; the 48 tensors of a small pair of networks in 7 us, behind the 3 us of the coefficients.
#include "common.hpp"
#include "elem.hpp"

using namespace nerfhip;

namespace {

constexpr int THREADS = 256, PER = 8, CHUNK = THREADS * PER;      // a workgroup's elements; 16 lanes hold a block of 128
constexpr int MAX_CHUNKS = 0xffffff;      // a launch holds fewer than 2^32 threads
constexpr int BATCH = NERF_ADAMW_BATCH;
static_assert(BATCH <= 64, "the tensor of a chunk is found with one ballot");

struct Tensors {
    void* p[BATCH];
    const void* g[BATCH];
    void* m[BATCH];
    void* v[BATCH];
    float* scale[BATCH];      // 8-bit states: sm, sv per block
    float* master[BATCH];     // 16-bit parameters
    int64_t count[BATCH];
    int first[BATCH];         // first chunk of every tensor among all chunks of the launch (INT_MAX behind the last)
};
static_assert(sizeof(Tensors) <= 3840, "kernel arguments are limited to 4 KB");

struct Coef { float step_size, inv_sqrt_bc2, lr_wd; unsigned t; };

struct Steps { float* step[BATCH]; };

// steps += 1, and what follows from the count, in fp64
__global__ void __launch_bounds__(64) k_adamw_begin(int n, Steps s, const float* lr_dev, double lr, double beta1, double beta2, double wd,
                                                    Coef* __restrict__ coef) {
    const int i = threadIdx.x;
    if (i >= n) return;
    const float t = *s.step[i] + 1.0f;
    *s.step[i] = t;
    if (lr_dev) lr = (double)*lr_dev;
    Coef c;
    c.step_size = (float)(lr / (1.0 - pow(beta1, (double)t)));
    c.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
    c.lr_wd = (float)(lr * wd);
    c.t = (unsigned)t;
    coef[i] = c;
}

// 32 random bits of (element, step): a multiplicative hash finished by two rounds of xor-shift and multiply (the 32-bit finaliser
// published by C. Wellons as lowbias32)
__device__ __forceinline__ unsigned noise(int64_t i, unsigned t) {
    unsigned h = (unsigned)i * 0x9E3779B1u + (unsigned)(i >> 32) * 0xC2B2AE3Du + t * 0x85EBCA77u;
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h *= 0x846CA68Bu;
    return h ^ (h >> 16);
}

// 0 <= u <= 448 -> e4m3, rounded up when the remainder of a grid step and r / 65536 reach a whole one
__device__ __forceinline__ unsigned to_e4m3(float u, unsigned r) {
    const unsigned normal = ((__float_as_uint(u) + (r << 4)) >> 20) - (120u << 3);
    const unsigned low = (unsigned)(u * 512.0f + (float)r * (1.0f / 65536.0f));
    return u < 0x1p-6f ? low : normal;
}
// 0 <= u <= 57344 -> e5m2 likewise
__device__ __forceinline__ unsigned to_e5m2(float u, unsigned r) {
    const unsigned normal = ((__float_as_uint(u) + (r << 5)) >> 21) - (112u << 2);
    const unsigned low = (unsigned)(u * 65536.0f + (float)r * (1.0f / 65536.0f));
    return u < 0x1p-14f ? low : normal;
}

// largest over the 16 lanes of a row, on the bits of non-negative floats: a NaN is larger than every number and stays
template <int CTRL>
__device__ __forceinline__ unsigned max_ror(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
    return o > v ? o : v;
}
__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = max_ror<0x121>(v);      // row_ror:1, 2, 4, 8
    v = max_ror<0x122>(v);
    v = max_ror<0x124>(v);
    return max_ror<0x128>(v);
}

template <typename T>
__device__ __forceinline__ void fetch(const T* p, int left, float (&out)[PER]) {
    if (left >= PER) {
        load_vec<T, PER>(p, out);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) out[e] = e < left ? (float)p[e] : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void put(T* p, int left, const float (&in)[PER]) {
    if (left >= PER) {
        store_vec<T, PER>(p, in);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (e < left) p[e] = (T)in[e];
    }
}
__device__ __forceinline__ void fetch_codes(const uint8_t* p, int left, unsigned (&w)[2]) {
    if (left >= PER) {
        __builtin_memcpy(w, p, PER);
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (e < left) w[e >> 2] |= (unsigned)p[e] << (8 * (e & 3));
    }
}
__device__ __forceinline__ void put_codes(uint8_t* p, int left, const unsigned (&w)[2]) {
    if (left >= PER) {
        __builtin_memcpy(p, w, PER);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (e < left) p[e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
}

template <typename T, bool EIGHT>
__global__ void __launch_bounds__(THREADS) k_adamw(Tensors ts, const Coef* __restrict__ coef, float w1, float w2, float eps) {
    constexpr bool NARROW = sizeof(T) == 2;
    const int lane = threadIdx.x & 63;
    const int chunk = (int)blockIdx.x;
    const int i = __builtin_popcountll(__ballot(lane < BATCH && ts.first[lane < BATCH ? lane : 0] <= chunk)) - 1;
    const Coef c = coef[i];
    const int64_t e0 = (int64_t)(chunk - ts.first[i]) * CHUNK + threadIdx.x * PER;
    const int64_t rest = ts.count[i] - e0;
    const int left = rest > PER ? PER : (rest < 0 ? 0 : (int)rest);
    T* pp = (T*)ts.p[i] + e0;
    const T* gp = (const T*)ts.g[i] + e0;
    float* masterp = NARROW ? ts.master[i] + e0 : nullptr;

    float p[PER], g[PER], m[PER], v[PER];
    fetch<T>(gp, left, g);
    fetch<T>(pp, left, p);
    if (NARROW) {     // the master copy, unless the parameter was written since it was rounded from it
        float master[PER];
        fetch<float>(masterp, left, master);
#pragma unroll
        for (int e = 0; e < PER; ++e) p[e] = (float)(T)master[e] == p[e] ? master[e] : p[e];
    }
    const int64_t block = (e0 >> 7);
    float *mp = nullptr, *vp = nullptr;
    uint8_t *mc = nullptr, *vc = nullptr;
    if (EIGHT) {
        mc = (uint8_t*)ts.m[i] + e0;
        vc = (uint8_t*)ts.v[i] + e0;
        unsigned a[2], b[2];
        fetch_codes(mc, left, a);
        fetch_codes(vc, left, b);
        float sm = 0.0f, sv = 0.0f;
        if (left > 0) {
            sm = ts.scale[i][2 * block];
            sv = ts.scale[i][2 * block + 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(a[h], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(a[h], true);
            const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8(b[h], false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8(b[h], true);
            m[4 * h] = m01[0] * sm; m[4 * h + 1] = m01[1] * sm; m[4 * h + 2] = m23[0] * sm; m[4 * h + 3] = m23[1] * sm;
            v[4 * h] = v01[0] * sv; v[4 * h + 1] = v01[1] * sv; v[4 * h + 2] = v23[0] * sv; v[4 * h + 3] = v23[1] * sv;
        }
    } else {
        mp = (float*)ts.m[i] + e0;
        vp = (float*)ts.v[i] + e0;
        fetch<float>(mp, left, m);
        fetch<float>(vp, left, v);
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        {      // (each operation rounded by itself: with states in 8 bits a last place can move a code by a whole step)
#pragma clang fp contract(off)
            m[e] = m[e] + w1 * (g[e] - m[e]);
            v[e] = v[e] + w2 * (g[e] * g[e] - v[e]);
        }
        const float denom = sqrtf(v[e]) * c.inv_sqrt_bc2 + eps;
        p[e] -= c.lr_wd * p[e] + c.step_size * m[e] / denom;
    }
    if (EIGHT) {
        unsigned am = 0, av = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            if (e >= left) continue;
            const unsigned mb = __float_as_uint(m[e]) & 0x7fffffffu, vb = __float_as_uint(v[e]) & 0x7fffffffu;
            am = mb > am ? mb : am;
            av = vb > av ? vb : av;
        }
        // (a scale is what the codes are divided by here and multiplied by in the next step: at least LEAST, unless all is 0)
        constexpr float LEAST = 1e-38f;
        am = row_max(am);
        av = row_max(av);
        float sm = __uint_as_float(am) * (1.0f / 448.0f), sv = __uint_as_float(av) * (1.0f / 57344.0f);
        if (am && sm < LEAST) sm = LEAST;      // (a NaN stays)
        if (av && sv < LEAST) sv = LEAST;
        const float dm = fmaxf(sm, LEAST), dv = fmaxf(sv, LEAST);
        unsigned a[2] = {0, 0}, b[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const unsigned h = noise(e0 + e, c.t);
            unsigned cm = to_e4m3(fminf(fabsf(m[e]) / dm, 448.0f), h & 0xffffu);
            cm |= (__float_as_uint(m[e]) >> 31) << 7;
            unsigned cv = to_e5m2(fminf(v[e] / dv, 57344.0f), h >> 16);
            if (cv == 0 && v[e] > 0.0f) cv = 1;
            a[e >> 2] |= cm << (8 * (e & 3));
            b[e >> 2] |= cv << (8 * (e & 3));
        }
        put_codes(mc, left, a);
        put_codes(vc, left, b);
        if (left > 0 && (threadIdx.x & 15) == 0) {
            ts.scale[i][2 * block] = sm;
            ts.scale[i][2 * block + 1] = sv;
        }
    } else {
        put<float>(mp, left, m);
        put<float>(vp, left, v);
    }
    if (NARROW) put<float>(masterp, left, p);
    put<T>(pp, left, p);
}

}  // namespace

extern "C" {

int64_t nerf_adamw_workspace_floats(int n_tensors) { return (int64_t)(n_tensors < 0 ? 0 : n_tensors) * 4; }

int nerf_adamw_step(int n_tensors, const int64_t* counts, int type, int state_bits, void* const* params, const void* const* grads,
                    void* const* exp_avg, void* const* exp_avg_sq, float* const* scales, float* const* masters, float* const* steps,
                    const float* lr_dev, double lr, double beta1, double beta2, double eps, double weight_decay, float* workspace,
                    void* stream_) {
    NERF_REQUIRE(n_tensors >= 0, "nerf_adamw_step: n_tensors=%d", n_tensors);
    NERF_REQUIRE(elem_type_ok(type), "nerf_adamw_step: type=%d", type);
    NERF_REQUIRE(state_bits == 32 || state_bits == 8, "nerf_adamw_step: state_bits=%d is neither 32 nor 8", state_bits);
    NERF_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && weight_decay >= 0.0,
                 "nerf_adamw_step: beta1=%g beta2=%g eps=%g weight_decay=%g", beta1, beta2, eps, weight_decay);
    if (n_tensors == 0) return 0;
    const bool eight = state_bits == 8, narrow = type != NERF_F32;
    NERF_REQUIRE(counts && params && grads && exp_avg && exp_avg_sq && steps && workspace && (!eight || scales) && (!narrow || masters),
                 "nerf_adamw_step: null pointer");
    for (int i = 0; i < n_tensors; ++i) {
        NERF_REQUIRE(counts[i] >= 0 && counts[i] <= (int64_t)CHUNK * MAX_CHUNKS, "nerf_adamw_step: counts[%d]=%lld", i, (long long)counts[i]);
        NERF_REQUIRE(steps[i], "nerf_adamw_step: no step counter for tensor %d", i);
        NERF_REQUIRE(counts[i] == 0 || (params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i] && (!eight || scales[i]) && (!narrow || masters[i])),
                     "nerf_adamw_step: null pointer in tensor %d", i);
    }
    hipStream_t stream = as_stream(stream_);
    for (int a = 0; a < n_tensors;) {
        // as many tensors as one launch's table and grid hold
        Tensors ts{};
        Steps st{};
        int n = 0;
        int64_t chunks = 0;
        while (a + n < n_tensors && n < BATCH) {
            const int64_t more = (counts[a + n] + CHUNK - 1) / CHUNK;
            if (chunks + more > MAX_CHUNKS) break;      // (a tensor alone fits: checked above)
            const int i = a + n;
            ts.p[n] = params[i]; ts.g[n] = grads[i]; ts.m[n] = exp_avg[i]; ts.v[n] = exp_avg_sq[i];
            ts.scale[n] = eight ? scales[i] : nullptr;
            ts.master[n] = narrow ? masters[i] : nullptr;
            ts.count[n] = counts[i];
            ts.first[n] = (int)chunks;
            st.step[n] = steps[i];
            chunks += more;
            ++n;
        }
        for (int k = n; k < BATCH; ++k) ts.first[k] = 0x7fffffff;
        Coef* coef = reinterpret_cast<Coef*>(workspace) + a;
        hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(64), 0, stream, n, st, lr_dev, lr, beta1, beta2, weight_decay, coef);
        int rc = launched("nerf_adamw_step (counts)");
        if (rc) return rc;
        if (chunks > 0) {
            const float w1 = (float)(1.0 - beta1), w2 = (float)(1.0 - beta2);
#define GO(T, E) hipLaunchKernelGGL((k_adamw<T, E>), dim3((unsigned)chunks), dim3(THREADS), 0, stream, ts, coef, w1, w2, (float)eps)
            if (type == NERF_F32) { if (eight) GO(float, true); else GO(float, false); }
            else if (type == NERF_BF16) { if (eight) GO(bf16_t, true); else GO(bf16_t, false); }
            else { if (eight) GO(f16_t, true); else GO(f16_t, false); }
#undef GO
            rc = launched("nerf_adamw_step");
            if (rc) return rc;
        }
        a += n;
    }
    return 0;
}

}  // extern "C"
