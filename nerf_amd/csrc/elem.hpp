// Element types of the layer and optimiser operators (fp32, bf16, fp16): what is read is widened to fp32, what is written is
// rounded to nearest even once.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <cstdint>

namespace nerfhip {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline bool elem_type_ok(int type) { return type >= 0 && type <= 2; }

// N consecutive elements from any element's address: the memory system takes vector accesses at any alignment, so that odd strides and
// slices of larger buffers need no path of their own
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose { T e __attribute__((ext_vector_type(N))); };

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[N]) {
    const Loose<T, N> v = *reinterpret_cast<const Loose<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)v.e[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[N]) {
    Loose<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = (T)in[i];
    *reinterpret_cast<Loose<T, N>*>(p) = v;
}

}  // namespace nerfhip
