// Parts of the gated feed-forward block's kernels (gated_ffn.cu, gated_ffn_map.cuh): activations on pairs of values, the
// 32 x 32 staging tiles between accumulators and tensor copies, tensor maps.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "fh_kernels.h"
#include "row_ops.cuh"
#include "umma_tile.cuh"

using namespace rows;

namespace {

constexpr int kMaxChannels = 1 << 20;
constexpr int kSms = 148;

__device__ unsigned long long g_ffn_timeouts;

#define FH_TRY(call)                              \
    do {                                          \
        const cudaError_t e_ = (call);            \
        if (e_ != cudaSuccess) return e_;         \
    } while (0)

// ---- activations ----

__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// s = 1 / (1 + exp(-z)) of a pair, with one reciprocal for both (the special functions' unit is what bounds the narrow cases):
// 1 / a = b / (a b). The powers stop at 2^60 so that their product stays finite; beyond (z < -41) s is 0. c = 1 - s is formed as
// exp(-z) s: a difference would leave the reciprocal's error of 6e-8 where s is 1, which a derivative multiplies by g^3.
__device__ __forceinline__ float2 sigmoid2(float2 z, float2* c = nullptr) {
    const float2 t = mul2(z, pair(-1.44269504f));  // -log2(e) z
    const float2 e = make_float2(ex2(fminf(t.x, 60.0f)), ex2(fminf(t.y, 60.0f))), d = add2(e, pair(1.0f));
    const float2 s = mul2(pair(rcp(d.x * d.y)), make_float2(d.y, d.x));
    if (c) *c = mul2(e, s);
    return make_float2(t.x > 60.0f ? 0.0f : s.x, t.y > 60.0f ? 0.0f : s.y);
}
// Phi(g) = erfc(-g / sqrt 2) / 2 and exp(-g^2 / 2), by formula 7.1.26 of Abramowitz and Stegun (erfc to 1.5e-7): with
// z = |g| / sqrt 2 and t = 1 / (1 + p z), erfc(z) = t (a1 + t (a2 + ... + t a5)) exp(-z^2)
__device__ __forceinline__ void normal2(float2 g, float2& cdf, float2& e) {
    const float2 z = make_float2(fabsf(g.x), fabsf(g.y));
    const float2 d = fma2(z, pair(0.3275911f * 0.70710678f), pair(1.0f)), q = mul2(mul2(g, g), pair(-0.72134752f));
    const float2 t = make_float2(rcp(d.x), rcp(d.y));
    e = make_float2(ex2(q.x), ex2(q.y));
    float2 s = fma2(t, pair(1.061405429f), pair(-1.453152027f));
    s = fma2(t, s, pair(1.421413741f));
    s = fma2(t, s, pair(-0.284496736f));
    s = fma2(t, s, pair(0.254829592f));
    s = mul2(mul2(mul2(s, t), e), pair(0.5f));  // erfc(z) / 2
    cdf = make_float2(g.x < 0.0f ? s.x : 1.0f - s.x, g.y < 0.0f ? s.y : 1.0f - s.y);
}
// What keeps a NaN gate one where act(g) is no product with g: relu, and sigmoid2's value (the smallest of (NaN, 60) there is 60, so
// that a NaN does not reach the pair's other value)
__device__ __forceinline__ float2 relu2(float2 g) { return make_float2(g.x <= 0.0f ? 0.0f : g.x, g.y <= 0.0f ? 0.0f : g.y); }
__device__ __forceinline__ float2 keep_nan(float2 g, float2 s) { return make_float2(g.x != g.x ? g.x : s.x, g.y != g.y ? g.y : s.y); }
// act(g) of a pair. 0.5 (1 + tanh z) = sigmoid(2 z), so the tanh form of gelu is g sigmoid(2 sqrt(2 / pi) (g + 0.044715 g^3))
template <int ACT>
__device__ __forceinline__ float2 act_of(float2 g) {
    if (ACT == FH_ACT_RELU) return relu2(g);
    if (ACT == FH_ACT_GELU) {
        float2 cdf, e;
        normal2(g, cdf, e);
        return mul2(g, cdf);
    }
    float2 z = g;
    if (ACT == FH_ACT_GELU_TANH) z = mul2(g, fma2(mul2(g, g), pair(0.07135481f), pair(1.59576912f)));
    const float2 s = sigmoid2(z);
    return ACT == FH_ACT_SIGMOID ? keep_nan(g, s) : mul2(g, s);
}
// act(g) and its derivative (relu's is 1 where g > 0, so 0 at a NaN)
template <int ACT>
__device__ __forceinline__ void act_both(float2 g, float2& v, float2& dv) {
    if (ACT == FH_ACT_RELU) {
        v = relu2(g);
        dv = make_float2(g.x > 0.0f ? 1.0f : 0.0f, g.y > 0.0f ? 1.0f : 0.0f);
    } else if (ACT == FH_ACT_GELU) {
        float2 cdf, e;
        normal2(g, cdf, e);
        v = mul2(g, cdf);
        dv = fma2(mul2(g, pair(0.39894228f)), e, cdf);
    } else {
        // g^2 of the derivative's polynomial is held finite, since 1 - s is 0 before it could matter
        const float2 g2 = mul2(g, g), g2f = make_float2(fminf(g2.x, 1e30f), fminf(g2.y, 1e30f));
        float2 z = g, c;
        if (ACT == FH_ACT_GELU_TANH) z = mul2(g, fma2(g2, pair(0.07135481f), pair(1.59576912f)));
        const float2 s = sigmoid2(z, &c);  // c: 1 - s
        if (ACT == FH_ACT_SIGMOID) {
            v = keep_nan(g, s);
            dv = mul2(v, c);
        } else {
            v = mul2(g, s);
            // s + g s (1 - s) dz / dg
            const float2 w = mul2(v, c);
            dv = ACT == FH_ACT_SILU ? add2(s, w) : fma2(w, fma2(g2f, pair(0.21406443f), pair(1.59576912f)), s);
        }
    }
}

// ---- staging tiles ----

constexpr int kTile = 32 * 64;  // a tail's staging tile: 32 rows of 32 columns, 64-byte swizzled

// 16 columns (half h of 32) of this lane's row of a staging tile: chunk c of a row lies at c ^ (row / 2 % 4)
__device__ __forceinline__ uint32_t tile_at(uint32_t tile, int lane, int h, int c) {
    return tile + lane * 64 + (((2 * h + c) ^ ((lane >> 1) & 3)) << 4);
}
template <typename T>
__device__ __forceinline__ void tile_put(uint32_t tile, int lane, int h, const float2 (&v)[8]) {
#pragma unroll
    for (int c = 0; c < 2; c++)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(tile_at(tile, lane, h, c)), "r"(Elem<T>::from2(v[4 * c].x, v[4 * c].y)),
                     "r"(Elem<T>::from2(v[4 * c + 1].x, v[4 * c + 1].y)), "r"(Elem<T>::from2(v[4 * c + 2].x, v[4 * c + 2].y)),
                     "r"(Elem<T>::from2(v[4 * c + 3].x, v[4 * c + 3].y))
                     : "memory");
}
// 16 columns in f32 are a staging tile of the same size and swizzle
__device__ __forceinline__ void tile_put32(uint32_t tile, int lane, const float2 (&v)[8]) {
#pragma unroll
    for (int c = 0; c < 4; c++)
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(tile_at(tile, lane, 0, c)), "f"(v[2 * c].x), "f"(v[2 * c].y),
                     "f"(v[2 * c + 1].x), "f"(v[2 * c + 1].y)
                     : "memory");
}
__device__ __forceinline__ void tile_get32(uint32_t tile, int lane, float2 (&v)[8]) {
#pragma unroll
    for (int c = 0; c < 4; c++)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                     : "=f"(v[2 * c].x), "=f"(v[2 * c].y), "=f"(v[2 * c + 1].x), "=f"(v[2 * c + 1].y)
                     : "r"(tile_at(tile, lane, 0, c))
                     : "memory");
}
__device__ __noinline__ void tile_out32(uint32_t tile, int lane, float* p, int valid) {
    for (int i = 0; i < valid; i++) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(tile_at(tile, lane, 0, i >> 2) + 4 * (i & 3)) : "memory");
        p[i] = v;
    }
}
// this lane's row of a staging tile, `valid` columns of it, to p: in place of a tensor copy, which writes whole 16-byte
// pieces, where the output's columns end inside one
template <typename T>
__device__ __noinline__ void tile_out(uint32_t tile, int lane, T* p, int valid) {
    for (int c = 0; 8 * c < valid; c++) {
        uint4 q;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                     : "r"(tile_at(tile, lane, 0, c))
                     : "memory");
        store_chunk(p + 8 * c, valid - 8 * c, unpack<T>(q));
    }
}
// 2 N columns of a bias (the same for all lanes) as they lie in memory, 0 past `cols` and where there is none
template <typename T, int N>
__device__ __forceinline__ void load_bias(const void* bias, int c, int cols, uint32_t (&q)[N]) {
    const T* p = static_cast<const T*>(bias) + c;
    if (bias && c + 2 * N <= cols) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 t = reinterpret_cast<const uint4*>(p)[i];
            q[4 * i] = t.x, q[4 * i + 1] = t.y, q[4 * i + 2] = t.z, q[4 * i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            q[i] = Elem<T>::from2(bias && c + 2 * i < cols ? Elem<T>::to(p[2 * i]) : 0.0f,
                                  bias && c + 2 * i + 1 < cols ? Elem<T>::to(p[2 * i + 1]) : 0.0f);
    }
}
// 16 accumulators as pairs, and a bias added to them
__device__ __forceinline__ void pairs(const uint32_t* r, float2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}
template <typename T>
__device__ __forceinline__ void add_bias(const uint32_t* q, float2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = add2(v[i], Elem<T>::to2(q[i]));
}
template <int ACT>
__device__ __forceinline__ void glu16(const float2 (&g)[8], const float2 (&u)[8], float2 (&a)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = mul2(act_of<ACT>(g[i]), u[i]);
}
// g and u become dg and du, a = act(g) u (a may be da)
template <int ACT>
__device__ __forceinline__ void glu_grad16(const float2 (&da)[8], float2 (&g)[8], float2 (&u)[8], float2 (&a)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float2 v, dv;
        act_both<ACT>(g[i], v, dv);
        g[i] = mul2(mul2(da[i], u[i]), dv);
        const float2 d = mul2(da[i], v);
        a[i] = mul2(v, u[i]);
        u[i] = d;
    }
}

// ---- tensor maps ----

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

struct Matrix {  // [rows][cols] of 16-bit elements
    const void* p;
    long long pitch;
    long long rows;
    int cols;
};

// boxes of 64 columns x `box` rows, 128-byte swizzled (operands), or of 32 rows of 64 bytes, 64-byte swizzled (box 0: the tails;
// f32 with dtype kF32)
constexpr int kF32 = -1;
cudaError_t map_of(CUtensorMap* map, const Matrix& x, int box, int dtype) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)x.cols, (cuuint64_t)x.rows}, strides[1] = {(cuuint64_t)x.pitch * (dtype == kF32 ? 4 : 2)};
    const cuuint32_t boxes[2] = {box ? 64u : dtype == kF32 ? 16u : 32u, box ? (cuuint32_t)box : 32u}, one[2] = {1, 1};
    const CUresult r = fn(map, dtype == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == FH_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                          const_cast<void*>(x.p), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          box ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace
