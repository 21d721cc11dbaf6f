// Loads and stores of V consecutive elements of a storage type (float, half, bfloat16) as floats: one transaction of
// V * sizeof(T) bytes, whose address is a multiple of that size (V = 1 has no alignment beyond the type's).  Arithmetic
// is always in 32 bits; a store rounds once, to nearest.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dsb {

template <int BYTES> struct RawVec;
template <> struct RawVec<2> { typedef unsigned short type; };
template <> struct RawVec<4> { typedef unsigned int type; };
template <> struct RawVec<8> { typedef uint2 type; };
template <> struct RawVec<16> { typedef uint4 type; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T, int V> struct alignas(V == 3 ? sizeof(T) : V * sizeof(T)) Pack { T e[V]; };   // three go one by one

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    if constexpr (V == 3) return {{p[0], p[1], p[2]}};
    else {
    typedef typename RawVec<V * sizeof(T)>::type Raw;
    const Raw raw = *reinterpret_cast<const Raw*>(p);
    Pack<T, V> out;
    static_assert(sizeof(out) == sizeof(raw), "one transaction");
    memcpy(&out, &raw, sizeof(raw));
    return out;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_floats(T* p, const float (&v)[V]) {
    if constexpr (V == 3) {
#pragma unroll
        for (int i = 0; i < V; ++i) from_float(v[i], p[i]);
    } else {
    typedef typename RawVec<V * sizeof(T)>::type Raw;
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) from_float(v[i], out.e[i]);
    Raw raw;
    memcpy(&raw, &out, sizeof(raw));
    *reinterpret_cast<Raw*>(p) = raw;
    }
}

// The same under a condition, with only the store itself left out.
template <typename T, int V>
__device__ __forceinline__ void store_floats_if(T* p, const float (&v)[V], bool there) {
    if constexpr (V == 3) {
#pragma unroll
        for (int i = 0; i < V; ++i) if (there) from_float(v[i], p[i]);
    } else {
    typedef typename RawVec<V * sizeof(T)>::type Raw;
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) from_float(v[i], out.e[i]);
    Raw raw;
    memcpy(&raw, &out, sizeof(raw));
    if (there) *reinterpret_cast<Raw*>(p) = raw;
    }
}

// Calls f with a value of the storage type that `dtype` (DSB_DTYPE_*) names; false for an unknown one.
template <typename F>
bool with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case DSB_DTYPE_F32: f(float{}); return true;
        case DSB_DTYPE_F16: f(__half{}); return true;
        case DSB_DTYPE_BF16: f(__nv_bfloat16{}); return true;
        default: return false;
    }
}
inline int dtype_bytes(int dtype) { return dtype == DSB_DTYPE_F32 ? 4 : 2; }

}  // namespace dsb
