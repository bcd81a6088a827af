// Floating element types of the decoder operators: float, _Float16 and __bf16, read and written
// eight at a time at whatever alignment the caller's strides give.
#pragma once

#include "icx_common.hpp"

namespace icx {

inline bool is_float_kind(int dt) { return dt == ICX_F32 || dt == ICX_F16 || dt == ICX_BF16; }
inline size_t float_size(int dt) { return dt == ICX_F32 ? 4 : 2; }

// N elements at p (any alignment a T may have) as float.
template <int N, typename T>
__device__ __forceinline__ void load_f32(const T* p, float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec w;
    __builtin_memcpy(&w, p, sizeof(T) * N);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)w[i];
}

// float to T rounds to nearest even; past T's range it is an infinity.
template <int N, typename T>
__device__ __forceinline__ void store_f32(T* p, const float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec w;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (T)v[i];
    __builtin_memcpy(p, &w, sizeof(T) * N);
}

// Calls f with a null pointer of the element type that dt names.
template <typename F>
int with_float_type(int dt, F f) {
    if (dt == ICX_F32) return f((float*)nullptr);
    if (dt == ICX_F16) return f((_Float16*)nullptr);
    return f((__bf16*)nullptr);
}

}  // namespace icx
