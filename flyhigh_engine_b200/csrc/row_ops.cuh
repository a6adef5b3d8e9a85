// Helpers of the row operators (gated_ffn.cu, residual_norm.cu): element types, 16-byte chunks of a row, argument checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fh_kernels.h"

namespace rows {

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float2 to2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
    static __device__ __forceinline__ uint32_t from2(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float2 to2(uint32_t v) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    }
    static __device__ __forceinline__ uint32_t from2(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// 8 elements of a row as 4 pairs: arithmetic on pairs is one instruction for two elements
struct Chunk {
    float2 v[4];
    __device__ __forceinline__ float get(int i) const { return i & 1 ? v[i / 2].y : v[i / 2].x; }
    __device__ __forceinline__ void set(int i, float x) { (i & 1 ? v[i / 2].y : v[i / 2].x) = x; }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(0.0f, 0.0f);
    }
    // the elements from `valid` on become 0
    __device__ __forceinline__ void cut(int valid) {
        if (valid >= 8) return;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= valid) set(i, 0.0f);
    }
};
template <typename T>
__device__ __forceinline__ Chunk unpack(const uint4& q) {
    return {{Elem<T>::to2(q.x), Elem<T>::to2(q.y), Elem<T>::to2(q.z), Elem<T>::to2(q.w)}};
}
// 8 elements at p, `valid` of them inside the row; vec: p lies on a 16-byte boundary. A whole chunk on a boundary is one
// 16-byte access; else element by element, so that nothing past the row's channels is touched. The rest read as 0.
template <typename T>
__device__ __forceinline__ Chunk load_chunk(const T* p, int valid, bool vec = true) {
    if (valid >= 8 && vec) return unpack<T>(*reinterpret_cast<const uint4*>(p));
    Chunk c;
#pragma unroll
    for (int i = 0; i < 8; i++) c.set(i, i < valid ? Elem<T>::to(p[i]) : 0.0f);
    return c;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int valid, const Chunk& c, bool vec = true) {
    if (valid >= 8 && vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::from2(c.v[0].x, c.v[0].y), Elem<T>::from2(c.v[1].x, c.v[1].y),
                                                  Elem<T>::from2(c.v[2].x, c.v[2].y), Elem<T>::from2(c.v[3].x, c.v[3].y));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < valid) p[i] = Elem<T>::from(c.get(i));
    }
}

constexpr long long kMaxRows = (1ll << 31) - 256;

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// a tensor of `m` rows: present, aligned, its pitch a multiple of 8 that holds the channels (any pitch where it is empty)
inline bool good_rows(const void* p, long long pitch, int c, long long m) {
    if (m == 0) return true;
    return p && aligned16(p) && pitch >= c && (pitch & 7) == 0 && pitch < (1ll << 36);
}
// the same, or absent
inline bool good_rows_or_null(const void* p, long long pitch, int c, long long m) { return !p || good_rows(p, pitch, c, m); }

}  // namespace rows
