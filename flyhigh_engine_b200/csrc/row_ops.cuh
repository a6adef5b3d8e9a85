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

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Elem<T>::to2(w[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// 8 elements of a row, `valid` of them inside it (8: one 16-byte access; fewer: element by element, so that nothing
// past the row's channels is touched). The rest read as 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
    if (valid >= 8) {
        unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < valid ? Elem<T>::to(p[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[8]) {
    if (valid >= 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::from2(v[0], v[1]), Elem<T>::from2(v[2], v[3]),
                                                  Elem<T>::from2(v[4], v[5]), Elem<T>::from2(v[6], v[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < valid) p[i] = Elem<T>::from(v[i]);
    }
}

// the same for a row that may begin anywhere: `vec` where it is known to begin on a 16-byte boundary
template <typename T>
__device__ __forceinline__ void load8_any(const T* p, int valid, bool vec, float (&v)[8]) {
    if (vec) {
        load8(p, valid, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < valid ? Elem<T>::to(p[i]) : 0.0f;
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
