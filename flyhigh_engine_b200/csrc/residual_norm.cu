// The join of a block with its residual and the next block's norm (fhk_residual_norm) and its gradient.
//
//   y = x + s * gate * p, p = norm_post(f);  h = norm_pre(y);  norm(v) = n * w + b, n the normalised row
//
// Forward: one pass. LPR threads hold a row in registers (8 channels per chunk, NCH chunks per thread), so the mean,
// the variance (of the centred values, a second sum over registers) and the result need the row read once; x and f are
// read and y and h written once, which is the operator's floor: it is bound by HBM.
//
// Gradient: with d = dy + norm_pre'(dh) and q = s * gate * d,
//   norm'(dv) = r * (dn - n * mean(dn * n) [- mean(dn) for a layer norm]),  dn = dv * w
//   dx = d, df = norm_post'(q); dw_pre = sum dh * n_y, db_pre = sum dh.
// Every parameter gradient of the post side is formed from two column sums per gate row k, A1 = sum d * n_f and
// A0 = sum d: with Q = w A1 + b A0 (the column sum of d * p), dgate[k] = s Q[k], ds = sum_k gate[k] Q[k],
// dw_post = s sum_k gate[k] A1[k], db_post = s sum_k gate[k] A0[k]. So a thread keeps four sums per channel (two per
// side) for its columns over all rows of its CTA; a second kernel adds the CTAs' sums in a fixed order.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "fh_device.cuh"
#include "fh_kernels.h"
#include "launch.h"
#include "row_ops.cuh"

using namespace rows;

namespace {

constexpr int kMaxC = 8192;
constexpr int kForwardThreads = 1024, kGradThreads = 512;  // threads per SM that the registers are cut for

// the sum over the LPR threads that share a row, in a fixed order, returned to all of them. LPR <= 32: within a warp;
// above: over the CTA (LPR == its threads), red holding one float per warp and a buffer of its own for each call
// between two reuses.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = (LPR < 32 ? LPR : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (LPR > 32) {
        constexpr int NW = LPR / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = lane < NW ? red[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
// two sums at once
template <int LPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float* red) {
#pragma unroll
    for (int o = (LPR < 32 ? LPR : 32) / 2; o; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (LPR > 32) {
        constexpr int NW = LPR / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) reinterpret_cast<float2*>(red)[warp] = make_float2(a, b);
        __syncthreads();
        const float2 t = lane < NW ? reinterpret_cast<float2*>(red)[lane] : make_float2(0.0f, 0.0f);
        a = t.x;
        b = t.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
    }
    return make_float2(a, b);
}

// v -> its normalised row n (in place; channels outside the row stay 0, all of them where the thread has no row);
// returns 1 / the deviation.
// red: 3 x 64 floats (a sum's buffer is reused only after another sum's barrier)
template <int LPR, int NCH>
__device__ __forceinline__ float normalise(int kind, float (&v)[NCH][8], const int (&valid)[NCH], float inv_c, float eps,
                                           float* red) {
    float mean = 0.0f;
    if (kind == FH_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NCH; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) s += v[k][j];
        mean = row_sum<LPR>(s, red) * inv_c;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[k][j] = j < valid[k] ? v[k][j] - mean : 0.0f;
            q += v[k][j] * v[k][j];
        }
    const float r = 1.0f / sqrtf(row_sum<LPR>(q, red + 64) * inv_c + eps);
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) v[k][j] = j < valid[k] ? v[k][j] * r : 0.0f;
    return r;
}

template <typename T>
__device__ __forceinline__ void mul_vec(float (&v)[8], const void* w, long long at, int valid) {
    if (!w) return;
    float t[8];
    load8(static_cast<const T*>(w) + at, valid, t);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= t[j];
}
// by the gate's row, which may begin anywhere
template <typename T, typename P>
__device__ __forceinline__ void mul_gate(float (&v)[8], const P& p, long long at, int valid) {
    if (!p.gate) return;
    float t[8];
    load8_any(static_cast<const T*>(p.gate) + at, valid, (p.gate_pitch & 7) == 0 && ((uintptr_t)p.gate & 15) == 0, t);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= t[j];
}
template <typename T>
__device__ __forceinline__ void add_vec(float (&v)[8], const void* w, long long at, int valid) {
    if (!w) return;
    float t[8];
    load8(static_cast<const T*>(w) + at, valid, t);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += t[j];
}

// A thread's own ring of rows in shared memory: asynchronous 16-byte copies of its chunks, STAGES - 1 rows ahead. A thread
// reads back only what it copied, so no barrier is needed, and the rows in flight cost no registers. A chunk that is partly
// (or wholly) outside its row copies the elements inside it and the rest is zero.
template <typename T, int THREADS, int NCH, int TENSORS, int STAGES>
struct Ring {
    uint4* buf;
    static constexpr size_t kBytes = (size_t)STAGES * TENSORS * NCH * THREADS * 16;
    __device__ __forceinline__ uint4* slot(int stage, int tensor, int k) const {
        return buf + ((stage * TENSORS + tensor) * NCH + k) * THREADS + threadIdx.x;
    }
    __device__ __forceinline__ void copy(int stage, int tensor, int k, const T* base, long long at, int valid) const {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(slot(stage, tensor, k));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(valid > 0 ? base + at : base),
                     "r"(valid > 0 ? 2 * valid : 0)
                     : "memory");
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory"); }
    __device__ __forceinline__ void read(int stage, int tensor, int k, float (&v)[8]) const {
        unpack8<T>(*slot(stage, tensor, k), v);
    }
};

// THREADS / LPR rows at a time per CTA
template <typename T, int THREADS, int LPR, int NCH, int STAGES>
__global__ void __launch_bounds__(THREADS, kForwardThreads / THREADS) k_residual_norm(const FhResidualNormParams p, long long rows_per_gate) {
    __shared__ float red[4 * 64];
    extern __shared__ uint4 ring_mem[];
    const Ring<T, THREADS, NCH, 2, STAGES> ring{ring_mem};
    constexpr int RPC = THREADS / LPR;
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = max(0, min(8, p.c - 8 * (l + k * LPR)));
    const T* x = static_cast<const T*>(p.x);
    const T* f = static_cast<const T*>(p.f);
    const long long first = (long long)blockIdx.x * RPC + sub, step = (long long)gridDim.x * RPC;
    auto fetch = [&](long long row, int stage) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int vk = row < p.m ? valid[k] : 0, c = 8 * (l + k * LPR);
            ring.copy(stage, 0, k, x, row * p.x_pitch + c, vk);
            if (f) ring.copy(stage, 1, k, f, row * p.f_pitch + c, vk);
        }
        ring.commit();
    };
#pragma unroll
    for (int q = 0; q < STAGES - 1; q++) fetch(first + q * step, q);
    int stage = 0;
    // every thread of a CTA runs the same number of iterations: the sums are CTA-wide barriers or whole-warp shuffles
    for (long long row = first; row - sub < p.m; row += step) {
        const bool on = row < p.m;
        float xv[NCH][8], fv[NCH][8];
        int vr[NCH];  // the channels of this thread's row
        ring.wait();
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            vr[k] = on ? valid[k] : 0;
            ring.read(stage, 0, k, xv[k]);
            if (f) ring.read(stage, 1, k, fv[k]);
        }
        fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (f) {
            if (p.post != FH_NORM_NONE) normalise<LPR, NCH>(p.post, fv, vr, inv_c, p.eps, red);
            const long long grow = p.gate && on ? row / rows_per_gate * p.gate_pitch : 0;
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                const int c = 8 * (l + k * LPR);
                if (valid[k]) {
                    mul_vec<T>(fv[k], p.w_post, c, valid[k]);
                    add_vec<T>(fv[k], p.b_post, c, valid[k]);
                    mul_vec<T>(fv[k], p.scale, c, valid[k]);
                    mul_gate<T>(fv[k], p, grow + c, valid[k]);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) xv[k][j] += j < valid[k] ? fv[k][j] : 0.0f;
                if (p.y && on && valid[k]) store8(static_cast<T*>(p.y) + row * p.y_pitch + c, valid[k], xv[k]);
            }
        }
        if (p.h) {
            normalise<LPR, NCH>(p.pre, xv, vr, inv_c, p.eps, red + 128);
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                const int c = 8 * (l + k * LPR);
                if (!valid[k]) continue;
                mul_vec<T>(xv[k], p.w_pre, c, valid[k]);
                add_vec<T>(xv[k], p.b_pre, c, valid[k]);
                if (on) store8(static_cast<T*>(p.h) + row * p.h_pitch + c, valid[k], xv[k]);
            }
        }
        if (LPR > 32) __syncthreads();  // the sums' buffers are free again
    }
}

// dn -> the gradient of the row that n was normalised from
template <int LPR, int NCH>
__device__ __forceinline__ void normalise_grad(int kind, float (&dn)[NCH][8], const float (&n)[NCH][8], float r,
                                               float inv_c, float* red) {
    float s1 = 0.0f, s0 = 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            s1 += dn[k][j] * n[k][j];
            s0 += dn[k][j];
        }
    const float2 s = row_sum2<LPR>(s1, s0, red);
    const float m1 = s.x * inv_c, m0 = kind == FH_NORM_LAYER ? s.y * inv_c : 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) dn[k][j] = r * (dn[k][j] - n[k][j] * m1 - m0);
}

// How a gradient's rows are shared out. Gate rows are `groups` runs of `len` rows. With few of them each run is cut
// into `slices` and a CTA takes one slice; with many a CTA takes `per_cta` whole runs one after another and finishes
// their dgate rows itself (slices == 1).
struct Split {
    long long len;
    int groups, slices, per_cta, ctas;
    bool whole;  // CTAs finish their runs' dgate
};

// the CTA's column sums, part [cta][4][c]: (A1, A0), or with whole runs (sum gate A1, sum gate A0); then sum dh n_y, sum dh
template <typename T, int THREADS, int LPR, int NCH, int STAGES, bool WHOLE>
__global__ void __launch_bounds__(THREADS, kGradThreads / THREADS) k_residual_norm_grad(const FhResidualNormGradParams p, const Split sp,
                                                                 float* part) {
    constexpr int RPC = THREADS / LPR;
    __shared__ float red[6 * 64];
    __shared__ float fold[RPC > 1 ? THREADS * NCH * 8 : 1];
    extern __shared__ uint4 ring_mem[];
    const Ring<T, THREADS, NCH, 4, STAGES> ring{ring_mem};
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = max(0, min(8, p.c - 8 * (l + k * LPR)));
    const T* f = static_cast<const T*>(p.f);
    float a1[NCH][8], a0[NCH][8], b1[NCH][8], b0[NCH][8];
    float g1[WHOLE ? NCH : 1][8], g0[WHOLE ? NCH : 1][8];
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            a1[k][j] = a0[k][j] = b1[k][j] = b0[k][j] = 0.0f;
            if (WHOLE) g1[k][j] = g0[k][j] = 0.0f;
        }
    // v summed over the CTA's row groups (in order), returned to all of them
    auto over_rows = [&](float (&v)[8]) {
        if (RPC == 1) return;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) fold[(sub * 8 + j) * LPR + l] = v[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float s = 0.0f;
#pragma unroll 4
            for (int i = 0; i < RPC; i++) s += fold[(i * 8 + j) * LPR + l];
            v[j] = s;
        }
    };

    const int first = WHOLE ? blockIdx.x * sp.per_cta : blockIdx.x / sp.slices;
    const int last = WHOLE ? min(first + sp.per_cta, sp.groups) : first + 1;
    for (int grp = first; grp < last; grp++) {
        long long lo = (long long)grp * sp.len, hi = lo + sp.len;
        if (!WHOLE) {
            const int sl = blockIdx.x % sp.slices;
            const long long base = lo;
            lo = base + sp.len * sl / sp.slices;
            hi = base + sp.len * (sl + 1) / sp.slices;
        }
        auto fetch = [&](long long row, int stage) {
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                const int vk = row < hi ? valid[k] : 0, c = 8 * (l + k * LPR);
                if (p.dy) ring.copy(stage, 0, k, static_cast<const T*>(p.dy), row * p.dy_pitch + c, vk);
                if (p.dh) {
                    ring.copy(stage, 1, k, static_cast<const T*>(p.dh), row * p.dh_pitch + c, vk);
                    ring.copy(stage, 2, k, static_cast<const T*>(p.y), row * p.y_pitch + c, vk);
                }
                if (f) ring.copy(stage, 3, k, f, row * p.f_pitch + c, vk);
            }
            ring.commit();
        };
        if (WHOLE) asm volatile("cp.async.wait_all;\n" ::: "memory");  // the last run's copies, before their slots are reused
#pragma unroll
        for (int q = 0; q < STAGES - 1; q++) fetch(lo + sub + q * RPC, q);
        int stage = 0;
        for (long long row = lo + sub; row - sub < hi; row += RPC) {
            const bool on = row < hi;
            float d[NCH][8], dh[NCH][8], yv[NCH][8], fv[NCH][8];
            int vr[NCH];  // the channels of this thread's row
            ring.wait();
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                vr[k] = on ? valid[k] : 0;
                if (p.dy) {
                    ring.read(stage, 0, k, d[k]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) d[k][j] = 0.0f;
                }
                if (p.dh) {
                    ring.read(stage, 1, k, dh[k]);
                    ring.read(stage, 2, k, yv[k]);
                }
                if (f) ring.read(stage, 3, k, fv[k]);
            }
            fetch(row + (STAGES - 1) * RPC, stage == 0 ? STAGES - 1 : stage - 1);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            if (p.dh) {
                const float r = normalise<LPR, NCH>(p.pre, yv, vr, inv_c, p.eps, red);
#pragma unroll
                for (int k = 0; k < NCH; k++) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        b1[k][j] += dh[k][j] * yv[k][j];
                        b0[k][j] += dh[k][j];
                    }
                    if (valid[k]) mul_vec<T>(dh[k], p.w_pre, 8 * (l + k * LPR), valid[k]);
                }
                normalise_grad<LPR, NCH>(p.pre, dh, yv, r, inv_c, red + 128);
#pragma unroll
                for (int k = 0; k < NCH; k++)
#pragma unroll
                    for (int j = 0; j < 8; j++) d[k][j] += j < vr[k] ? dh[k][j] : 0.0f;
            }
            if (p.dx) {
#pragma unroll
                for (int k = 0; k < NCH; k++)
                    if (on && valid[k])
                        store8(static_cast<T*>(p.dx) + row * p.dx_pitch + 8 * (l + k * LPR), valid[k], d[k]);
            }
            if (f) {
                float r = 1.0f;
                if (p.post != FH_NORM_NONE) r = normalise<LPR, NCH>(p.post, fv, vr, inv_c, p.eps, red + 256);
                const long long grow = p.gate ? (long long)grp * p.gate_pitch : 0;
#pragma unroll
                for (int k = 0; k < NCH; k++) {
                    const int c = 8 * (l + k * LPR);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        a1[k][j] += d[k][j] * fv[k][j];
                        a0[k][j] += d[k][j];
                    }
                    if (valid[k]) {
                        mul_vec<T>(d[k], p.scale, c, valid[k]);
                        mul_gate<T>(d[k], p, grow + c, valid[k]);
                        mul_vec<T>(d[k], p.w_post, c, valid[k]);
                    }
                }
                if (p.df) {
                    if (p.post != FH_NORM_NONE) normalise_grad<LPR, NCH>(p.post, d, fv, r, inv_c, red + 128);
#pragma unroll
                    for (int k = 0; k < NCH; k++)
                        if (on && valid[k])
                            store8(static_cast<T*>(p.df) + row * p.df_pitch + 8 * (l + k * LPR), valid[k], d[k]);
                }
            }
            if (LPR > 32) __syncthreads();
        }
        if (WHOLE) {  // the run's dgate row, and its share of the sums over gate rows
            const long long grow = p.gate ? (long long)grp * p.gate_pitch : 0;
#pragma unroll
            for (int k = 0; k < (WHOLE ? NCH : 1); k++) {
                const int c = 8 * (l + k * LPR);
                over_rows(a1[k]);
                over_rows(a0[k]);
                if (valid[k] && sub == 0) {
                    if (p.dgate) {
                        float q[8], w0[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            q[j] = a1[k][j];
                            w0[j] = a0[k][j];
                        }
                        mul_vec<T>(q, p.w_post, c, valid[k]);
                        if (p.b_post) {
                            mul_vec<T>(w0, p.b_post, c, valid[k]);
#pragma unroll
                            for (int j = 0; j < 8; j++) q[j] += w0[j];
                        }
                        mul_vec<T>(q, p.scale, c, valid[k]);
                        T* dst = static_cast<T*>(p.dgate) + (long long)grp * p.dgate_pitch + c;
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (j < valid[k]) dst[j] = Elem<T>::from(q[j]);
                    }
                    mul_gate<T>(a1[k], p, grow + c, valid[k]);
                    mul_gate<T>(a0[k], p, grow + c, valid[k]);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    // every row group of the CTA holds the run's whole sum: the first keeps it
                    g1[k][j] += sub == 0 ? a1[k][j] : 0.0f;
                    g0[k][j] += sub == 0 ? a0[k][j] : 0.0f;
                    a1[k][j] = a0[k][j] = 0.0f;
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");

    // the CTA's sums
    float* out = part + (long long)blockIdx.x * 4 * p.c;
    auto put = [&](int q, float (&v)[NCH][8], bool summed) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            if (!summed) over_rows(v[k]);
            const int c = 8 * (l + k * LPR);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (sub == 0 && j < valid[k]) out[(long long)q * p.c + c + j] = v[k][j];
        }
    };
    if constexpr (WHOLE) {
        put(0, g1, true);
        put(1, g0, true);
    } else {
        put(0, a1, false);
        put(1, a0, false);
    }
    put(2, b1, false);
    put(3, b0, false);
}

// 32 columns per CTA and 32 warps over the CTAs' sums; blockIdx.y: 0 the post side, 1 the pre side. Up to 32 gate rows at a
// time, each one's CTAs shared out over 32 / rows warps, whose sums are added in order.
template <typename T>
__global__ void __launch_bounds__(1024) k_residual_norm_params(const FhResidualNormGradParams p, const Split sp,
                                                               const float* part) {
    pdl_wait();
    __shared__ float2 s[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const bool on = col < p.c, post = blockIdx.y == 0;
    auto at = [&](const void* v, long long i, float none) { return v && on ? Elem<T>::to(static_cast<const T*>(v)[i]) : none; };
    auto put = [&](void* v, long long i, float x) {
        if (v && on) static_cast<T*>(v)[i] = Elem<T>::from(x);
    };
    // the pre side and whole runs are one sum over all CTAs
    const int groups = post && !sp.whole ? sp.groups : 1, slices = sp.ctas / groups;
    const float wp = at(p.w_post, col, 1.0f), bp = at(p.b_post, col, 0.0f), sc = at(p.scale, col, 1.0f);
    float g1 = 0.0f, g0 = 0.0f;
    for (int k0 = 0; k0 < groups; k0 += 32) {
        const int batch = min(32, groups - k0), parts = 32 / batch;
        float2 v = make_float2(0.0f, 0.0f);
        if (on && warp < batch * parts) {
            const int k = k0 + warp / parts, q = warp % parts;
            const float* src = part + (post ? 0 : 2 * (long long)p.c) + col;
            const int lo = k * slices + slices * q / parts, hi = k * slices + slices * (q + 1) / parts;
#pragma unroll 8
            for (int i = lo; i < hi; i++) {
                v.x += src[(long long)i * 4 * p.c];
                v.y += src[(long long)i * 4 * p.c + p.c];
            }
        }
        __syncthreads();
        s[warp][lane] = v;
        __syncthreads();
        if (warp == 0)
            for (int b = 0; b < batch; b++) {
                float t1 = 0.0f, t0 = 0.0f;
                for (int q = 0; q < parts; q++) {
                    t1 += s[b * parts + q][lane].x;
                    t0 += s[b * parts + q][lane].y;
                }
                if (post && !sp.whole) {
                    const int k = k0 + b;
                    const float g = at(p.gate, (long long)k * p.gate_pitch + col, 1.0f);
                    if (p.gate) put(p.dgate, (long long)k * p.dgate_pitch + col, sc * (wp * t1 + bp * t0));
                    t1 *= g;
                    t0 *= g;
                }
                g1 += t1;
                g0 += t0;
            }
    }
    if (warp != 0) return;
    if (post) {
        put(p.dscale, col, wp * g1 + bp * g0);
        put(p.dw_post, col, sc * g1);
        put(p.db_post, col, sc * g0);
    } else {
        put(p.dw_pre, col, g1);
        put(p.db_pre, col, g0);
    }
}

constexpr int kSms = 148;

// allows a kernel its dynamic shared memory, once per device
template <typename K>
cudaError_t allow(K kernel, size_t bytes, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
        done[dev].store(true, std::memory_order_release);
    }
    return cudaSuccess;
}

template <typename T, int THREADS, int LPR, int NCH, int STAGES>
cudaError_t run_forward(const FhResidualNormParams& p, cudaStream_t st) {
    static std::atomic<bool> done[64];
    constexpr size_t smem = Ring<T, THREADS, NCH, 2, STAGES>::kBytes;
    const cudaError_t e = allow(k_residual_norm<T, THREADS, LPR, NCH, STAGES>, smem, done);
    if (e != cudaSuccess) return e;
    constexpr int RPC = THREADS / LPR;
    const long long want = (p.m + RPC - 1) / RPC;
    const int grid = (int)std::min<long long>(want, (long long)kSms * (kForwardThreads / THREADS));
    return fhk::launch(k_residual_norm<T, THREADS, LPR, NCH, STAGES>, dim3(grid), dim3(THREADS), smem, st, p,
                       p.gate ? p.m / p.gates : p.m);
}

template <typename T>
cudaError_t forward(const FhResidualNormParams& p, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    if (c8 <= 8) return run_forward<T, 256, 8, 1, 4>(p, st);
    if (c8 <= 32) return run_forward<T, 256, 32, 1, 4>(p, st);
    if (c8 <= 64) return run_forward<T, 256, 32, 2, 3>(p, st);
    if (c8 <= 128) return run_forward<T, 128, 128, 1, 4>(p, st);
    if (c8 <= 256) return run_forward<T, 128, 128, 2, 3>(p, st);
    if (c8 <= 512) return run_forward<T, 256, 256, 2, 3>(p, st);
    return run_forward<T, 512, 512, 2, 3>(p, st);
}

Split split_of(long long m, int c, int gates, bool gate) {
    Split s{};
    s.groups = gate ? gates : 1;
    s.len = m / s.groups;
    // as many CTAs as are resident at once: kGradThreads threads per SM in CTAs of 128, 256 or 512 (grad())
    const int target = kSms * (c > 2048 ? 1 : c > 1024 || c <= 256 ? 2 : 4);
    s.whole = s.groups > 1 && s.groups >= target;
    if (s.whole) {
        s.slices = 1;
        s.per_cta = (s.groups + target - 1) / target;
        s.ctas = (s.groups + s.per_cta - 1) / s.per_cta;
    } else {
        s.per_cta = 1;
        s.slices = (int)std::max<long long>(1, std::min<long long>(target / s.groups, s.len));
        s.ctas = s.groups * s.slices;
    }
    return s;
}

template <typename T, int THREADS, int LPR, int NCH, int STAGES, bool WHOLE>
cudaError_t run_grad_as(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    static std::atomic<bool> done[64];
    constexpr size_t smem = Ring<T, THREADS, NCH, 4, STAGES>::kBytes;
    const cudaError_t e = allow(k_residual_norm_grad<T, THREADS, LPR, NCH, STAGES, WHOLE>, smem, done);
    if (e != cudaSuccess) return e;
    return fhk::launch(k_residual_norm_grad<T, THREADS, LPR, NCH, STAGES, WHOLE>, dim3(sp.ctas), dim3(THREADS), smem, st, p, sp,
                       static_cast<float*>(p.scratch));
}
template <typename T, int THREADS, int LPR, int NCH, int STAGES>
cudaError_t run_grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    return sp.whole ? run_grad_as<T, THREADS, LPR, NCH, STAGES, true>(p, sp, st)
                    : run_grad_as<T, THREADS, LPR, NCH, STAGES, false>(p, sp, st);
}

template <typename T>
cudaError_t grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    cudaError_t e;
    if (c8 <= 8) e = run_grad<T, 256, 8, 1, 3>(p, sp, st);
    else if (c8 <= 32) e = run_grad<T, 256, 32, 1, 3>(p, sp, st);
    else if (c8 <= 128) e = run_grad<T, 128, 128, 1, 3>(p, sp, st);
    else if (c8 <= 256) e = run_grad<T, 256, 256, 1, 3>(p, sp, st);
    else if (c8 <= 512) e = run_grad<T, 512, 512, 1, 3>(p, sp, st);
    else e = run_grad<T, 512, 512, 2, 2>(p, sp, st);
    if (e != cudaSuccess) return e;
    const bool post = p.f && (p.dgate || p.dscale || p.dw_post || p.db_post), pre = p.dw_pre || p.db_pre;
    if (!post && !pre) return cudaSuccess;
    fhk::PdlScope pdl(true);  // it waits for the kernel above
    return fhk::launch(k_residual_norm_params<T>, dim3((p.c + 31) / 32, 2), dim3(1024), 0, st, p, sp,
                       static_cast<const float*>(p.scratch));
}

bool good_kind(int k) { return k == FH_NORM_NONE || k == FH_NORM_RMS || k == FH_NORM_LAYER; }

template <typename P>
bool good_common(const P* p) {
    if (p->m < 0 || p->m > kMaxRows || p->c < 1 || p->c > kMaxC || !good_kind(p->pre) || !good_kind(p->post)) return false;
    if (p->dtype != FH_F16 && p->dtype != FH_BF16) return false;
    if (!(p->eps >= 0.0f)) return false;
    if (p->gate ? (p->gates < 1 || p->m % p->gates != 0 || ((uintptr_t)p->gate & 1) || p->gate_pitch < p->c) : p->gates != 0)
        return false;
    return aligned16(p->scale) && aligned16(p->w_post) && aligned16(p->b_post) && aligned16(p->w_pre);
}

}  // namespace

extern "C" int fhk_residual_norm(const FhResidualNormParams* p, void* stream) {
    if (!p || !good_common(p) || !aligned16(p->b_pre)) return (int)cudaErrorInvalidValue;
    if (!good_rows(p->x, p->x_pitch, p->c, p->m)) return (int)cudaErrorInvalidValue;
    if (p->m > 0) {
        if ((p->f != nullptr) != (p->y != nullptr) || (p->pre != FH_NORM_NONE) != (p->h != nullptr)) return (int)cudaErrorInvalidValue;
        if (!p->f && (!p->h || p->gate || p->scale || p->post != FH_NORM_NONE)) return (int)cudaErrorInvalidValue;
    }
    if (!good_rows_or_null(p->f, p->f_pitch, p->c, p->m) || !good_rows_or_null(p->y, p->y_pitch, p->c, p->m) ||
        !good_rows_or_null(p->h, p->h_pitch, p->c, p->m))
        return (int)cudaErrorInvalidValue;
    if (p->m == 0) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return (int)(p->dtype == FH_F16 ? forward<__half>(*p, st) : forward<__nv_bfloat16>(*p, st));
}

extern "C" size_t fhk_residual_norm_grad_scratch_bytes(const FhResidualNormGradParams* p) {
    if (!p || p->m <= 0 || p->m > kMaxRows || p->c < 1 || p->c > kMaxC || p->gates < 0 || p->gates > p->m) return 0;
    return (size_t)split_of(p->m, p->c, p->gates, p->gates > 0).ctas * 4 * p->c * sizeof(float);
}

extern "C" int fhk_residual_norm_grad(const FhResidualNormGradParams* p, void* stream) {
    if (!p || !good_common(p)) return (int)cudaErrorInvalidValue;
    void* const vecs[5] = {p->dscale, p->dw_post, p->db_post, p->dw_pre, p->db_pre};
    for (const void* v : vecs)
        if (!aligned16(v)) return (int)cudaErrorInvalidValue;
    const bool pre = p->pre != FH_NORM_NONE;
    if (p->dh && !pre) return (int)cudaErrorInvalidValue;
    if ((p->dgate && !p->gate) || (p->dscale && !p->scale) || (p->dw_post && !p->w_post) || (p->dw_pre && !p->w_pre))
        return (int)cudaErrorInvalidValue;
    if (p->m > 0) {
        if (p->dh && !p->y) return (int)cudaErrorInvalidValue;
        if (!p->dy && !p->dh) return (int)cudaErrorInvalidValue;
        if (!p->f && (p->df || p->gate || p->scale || p->w_post || p->db_post || p->post != FH_NORM_NONE))
            return (int)cudaErrorInvalidValue;
    }
    if ((p->dw_pre || p->db_pre) && !pre) return (int)cudaErrorInvalidValue;
    if (!good_rows_or_null(p->dy, p->dy_pitch, p->c, p->m) || !good_rows_or_null(p->dh, p->dh_pitch, p->c, p->m) ||
        !good_rows_or_null(p->y, p->y_pitch, p->c, p->m) || !good_rows_or_null(p->f, p->f_pitch, p->c, p->m) ||
        !good_rows_or_null(p->dx, p->dx_pitch, p->c, p->m) || !good_rows_or_null(p->df, p->df_pitch, p->c, p->m) ||
        (p->dgate && (((uintptr_t)p->dgate & 1) || p->dgate_pitch < p->c)))
        return (int)cudaErrorInvalidValue;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->m == 0) {  // no rows: the parameters' gradients are zero
        const size_t row = 2 * (size_t)p->c;
        for (void* v : vecs)
            if (v) {
                const cudaError_t e = cudaMemsetAsync(v, 0, row, st);
                if (e != cudaSuccess) return (int)e;
            }
        if (p->dgate) return (int)cudaMemset2DAsync(p->dgate, 2 * (size_t)p->dgate_pitch, 0, row, (size_t)p->gates, st);
        return 0;
    }
    if (!p->scratch || !aligned16(p->scratch) || p->scratch_bytes < fhk_residual_norm_grad_scratch_bytes(p))
        return (int)cudaErrorInvalidValue;
    const Split sp = split_of(p->m, p->c, p->gates, p->gate != nullptr);
    return (int)(p->dtype == FH_F16 ? grad<__half>(*p, sp, st) : grad<__nv_bfloat16>(*p, sp, st));
}
