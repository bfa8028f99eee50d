// Eight consecutive elements of a row to and from fp32 registers, for fp32 / bf16 / fp16 storage.  Pointers
// need the alignment of one element only: the vector types below say so, and global memory instructions take
// any such address.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace nbx {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T>
struct Vec8 {   // 16-bit element types: one 16-byte access
    typedef T type __attribute__((ext_vector_type(8), aligned(2)));
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const typename Vec8<T>::type t = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    typename Vec8<T>::type t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
    *reinterpret_cast<typename Vec8<T>::type*>(p) = t;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    f32x4u a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = v[i];
        b[i] = v[4 + i];
    }
    *reinterpret_cast<f32x4u*>(p) = a;
    *reinterpret_cast<f32x4u*>(p + 4) = b;
}

// The first n (0 .. 8) of eight; the others read as 0 and are not written.
template <typename T>
__device__ __forceinline__ void load8n(const T* p, int n, float (&v)[8]) {
    if (n == 8) {
        load8(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8n(T* p, int n, const float (&v)[8]) {
    if (n == 8) {
        store8(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (T)v[i];
}

// Eight elements as loaded: nothing waits for them before unpack8.
template <typename T>
struct Raw8 {
    typename Vec8<T>::type v;
};
template <>
struct Raw8<float> {
    f32x4u a, b;
};
template <typename T>
__device__ __forceinline__ void fetch8n(const T* p, int n, Raw8<T>& r) {
    if (n == 8) {
        r.v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
}
__device__ __forceinline__ void fetch8n(const float* p, int n, Raw8<float>& r) {
    if (n == 8) {
        r.a = *reinterpret_cast<const f32x4u*>(p);
        r.b = *reinterpret_cast<const f32x4u*>(p + 4);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.a[i] = i < n ? p[i] : 0.f;
        r.b[i] = 4 + i < n ? p[4 + i] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r.v[i];
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = r.a[i];
        v[4 + i] = r.b[i];
    }
}

// Parameters: fp32, or the 16-bit type of the activations (code NBX_F32 / NBX_BF16 / NBX_F16, uniform).
__device__ __forceinline__ void load8p(const void* p, int dtype, int64_t at, int n, float (&v)[8]) {
    if (dtype == 0) load8n((const float*)p + at, n, v);
    else if (dtype == 1) load8n((const bf16*)p + at, n, v);
    else load8n((const f16*)p + at, n, v);
}
__device__ __forceinline__ void store1p(void* p, int dtype, int64_t at, float v) {
    if (dtype == 0) ((float*)p)[at] = v;
    else if (dtype == 1) ((bf16*)p)[at] = (bf16)v;
    else ((f16*)p)[at] = (f16)v;
}
__device__ __forceinline__ void store8p(void* p, int dtype, int64_t at, int n, const float (&v)[8]) {
    if (dtype == 0) store8n((float*)p + at, n, v);
    else if (dtype == 1) store8n((bf16*)p + at, n, v);
    else store8n((f16*)p + at, n, v);
}

// Sum over the 16 or 64 lanes that share a row, in every one of them.  Rotations within 16 lanes are operand
// modifiers of the add (no LDS permute); the four sixteens are then read as scalars.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
    static_assert(W == 16 || W == 64, "16 or 64 lanes");
    x = dpp_add<0x128>(x);   // row_ror:8, 4, 2, 1
    x = dpp_add<0x124>(x);
    x = dpp_add<0x122>(x);
    x = dpp_add<0x121>(x);
    if constexpr (W == 64) {
        const int i = __float_as_int(x);
        x = (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
            (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
    }
    return x;
}

}  // namespace nbx
