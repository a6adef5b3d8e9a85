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

#include "fh_device.cuh"
#include "fh_kernels.h"
#include "launch.h"
#include "row_ops.cuh"

using namespace rows;

namespace {

constexpr int kMaxC = 8192;

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

// THREADS / LPR rows at a time per CTA
template <typename T, int THREADS, int LPR, int NCH>
__global__ void __launch_bounds__(THREADS) k_residual_norm(const FhResidualNormParams p, long long rows_per_gate) {
    __shared__ float red[4 * 64];
    constexpr int RPC = THREADS / LPR;
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = max(0, min(8, p.c - 8 * (l + k * LPR)));
    const T* x = static_cast<const T*>(p.x);
    const T* f = static_cast<const T*>(p.f);
    // every thread of a CTA runs the same number of iterations: the sums are CTA-wide barriers or whole-warp shuffles
    for (long long r0 = (long long)blockIdx.x * RPC; r0 < p.m; r0 += (long long)gridDim.x * RPC) {
        const long long row = r0 + sub;
        const bool on = row < p.m;
        float xv[NCH][8], fv[NCH][8];
        int vr[NCH];  // the channels of this thread's row
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int vk = vr[k] = on ? valid[k] : 0, c = 8 * (l + k * LPR);
            load8(x + (vk ? row * p.x_pitch + c : 0), vk, xv[k]);
            if (f) load8(f + (vk ? row * p.f_pitch + c : 0), vk, fv[k]);
        }
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
template <typename T, int THREADS, int LPR, int NCH>
__global__ void __launch_bounds__(THREADS) k_residual_norm_grad(const FhResidualNormGradParams p, const Split sp,
                                                                 float* part) {
    constexpr int RPC = THREADS / LPR;
    __shared__ float red[6 * 64];
    __shared__ float fold[LPR > 32 ? 1 : RPC * LPR * NCH * 8];
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = max(0, min(8, p.c - 8 * (l + k * LPR)));
    const T* f = static_cast<const T*>(p.f);
    float a1[NCH][8], a0[NCH][8], g1[NCH][8], g0[NCH][8], b1[NCH][8], b0[NCH][8];
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) a1[k][j] = a0[k][j] = g1[k][j] = g0[k][j] = b1[k][j] = b0[k][j] = 0.0f;

    const int first = sp.whole ? blockIdx.x * sp.per_cta : blockIdx.x / sp.slices;
    const int last = sp.whole ? min(first + sp.per_cta, sp.groups) : first + 1;
    for (int grp = first; grp < last; grp++) {
        long long lo = (long long)grp * sp.len, hi = lo + sp.len;
        if (!sp.whole) {
            const int sl = blockIdx.x % sp.slices;
            const long long base = lo;
            lo = base + sp.len * sl / sp.slices;
            hi = base + sp.len * (sl + 1) / sp.slices;
        }
        for (long long r0 = lo; r0 < hi; r0 += RPC) {
            const long long row = r0 + sub;
            const bool on = row < hi;
            float d[NCH][8], dh[NCH][8], yv[NCH][8], fv[NCH][8];
            int vr[NCH];  // the channels of this thread's row
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                const int vk = vr[k] = on ? valid[k] : 0, c = 8 * (l + k * LPR);
                load8(static_cast<const T*>(p.dy) + (vk ? row * p.dy_pitch + c : 0), p.dy ? vk : 0, d[k]);
                if (p.dh) {
                    load8(static_cast<const T*>(p.dh) + (vk ? row * p.dh_pitch + c : 0), vk, dh[k]);
                    load8(static_cast<const T*>(p.y) + (vk ? row * p.y_pitch + c : 0), vk, yv[k]);
                }
                if (f) load8(f + (vk ? row * p.f_pitch + c : 0), vk, fv[k]);
            }
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
        if (sp.whole) {  // the run's dgate row, and its share of the sums over gate rows
            const long long grow = p.gate ? (long long)grp * p.gate_pitch : 0;
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                const int c = 8 * (l + k * LPR);
                float t1[8], t0[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    t1[j] = a1[k][j];
                    t0[j] = a0[k][j];
                    if (LPR <= 32 && RPC > 1) {  // rows of the CTA's other threads
                        for (int w = 0; w < 2; w++) {
                            __syncthreads();
                            fold[sub * LPR + l] = w ? t0[j] : t1[j];
                            __syncthreads();
                            float s = 0.0f;
                            for (int i = 0; i < RPC; i++) s += fold[i * LPR + l];
                            (w ? t0[j] : t1[j]) = s;
                        }
                    }
                    a1[k][j] = a0[k][j] = 0.0f;
                }
                if (!valid[k]) continue;
                if (p.dgate && sub == 0) {
                    float q[8], w0[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        q[j] = t1[j];
                        w0[j] = t0[j];
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
                mul_gate<T>(t1, p, grow + c, valid[k]);
                mul_gate<T>(t0, p, grow + c, valid[k]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    // every row group of the CTA holds the run's whole sum: only the first keeps it
                    g1[k][j] += sub == 0 ? t1[j] : 0.0f;
                    g0[k][j] += sub == 0 ? t0[j] : 0.0f;
                }
            }
        }
    }

    // the CTA's sums
    float* out = part + (long long)blockIdx.x * 4 * p.c;
#pragma unroll
    for (int q = 0; q < 4; q++) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int c = 8 * (l + k * LPR);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float v = q == 0 ? (sp.whole ? g1[k][j] : a1[k][j])
                          : q == 1 ? (sp.whole ? g0[k][j] : a0[k][j])
                          : q == 2 ? b1[k][j] : b0[k][j];
                if (LPR <= 32 && RPC > 1) {
                    __syncthreads();
                    fold[sub * LPR + l] = v;
                    __syncthreads();
                    if (sub == 0) {
                        v = 0.0f;
                        for (int i = 0; i < RPC; i++) v += fold[i * LPR + l];
                    }
                }
                if (sub == 0 && j < valid[k]) out[(long long)q * p.c + c + j] = v;
            }
        }
    }
}

// 32 columns per CTA, 8 threads per column over the CTAs' sums; blockIdx.y: 0 the post side, 1 the pre side
template <typename T>
__global__ void __launch_bounds__(256) k_residual_norm_params(const FhResidualNormGradParams p, const Split sp,
                                                              const float* part) {
    __shared__ float s1[8][33], s0[8][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
    const bool on = col < p.c;
    auto sum = [&](int lo, int hi, int which) -> float2 {  // over CTAs lo .. hi, to the threads of w == 0
        float v1 = 0.0f, v0 = 0.0f;
        if (on)
            for (int i = lo + w; i < hi; i += 8) {
                v1 += part[((long long)i * 4 + which) * p.c + col];
                v0 += part[((long long)i * 4 + which + 1) * p.c + col];
            }
        __syncthreads();
        s1[w][threadIdx.x & 31] = v1;
        s0[w][threadIdx.x & 31] = v0;
        __syncthreads();
        v1 = v0 = 0.0f;
        for (int i = 0; i < 8; i++) {
            v1 += s1[i][threadIdx.x & 31];
            v0 += s0[i][threadIdx.x & 31];
        }
        return make_float2(v1, v0);
    };
    auto at = [&](const void* v, long long i, float none) { return v && on ? Elem<T>::to(static_cast<const T*>(v)[i]) : none; };
    auto put = [&](void* v, long long i, float x) {
        if (v && on && w == 0) static_cast<T*>(v)[i] = Elem<T>::from(x);
    };
    if (blockIdx.y == 1) {
        const float2 b = sum(0, sp.ctas, 2);
        put(p.dw_pre, col, b.x);
        put(p.db_pre, col, b.y);
        return;
    }
    const float wp = at(p.w_post, col, 1.0f), bp = at(p.b_post, col, 0.0f), s = at(p.scale, col, 1.0f);
    float g1 = 0.0f, g0 = 0.0f;
    if (sp.whole) {
        const float2 a = sum(0, sp.ctas, 0);
        g1 = a.x;
        g0 = a.y;
    } else {
        for (int k = 0; k < sp.groups; k++) {
            const float2 a = sum(k * sp.slices, (k + 1) * sp.slices, 0);
            const float g = at(p.gate, (long long)k * p.gate_pitch + col, 1.0f);
            put(p.dgate, (long long)k * p.dgate_pitch + col, s * (wp * a.x + bp * a.y));
            g1 += g * a.x;
            g0 += g * a.y;
        }
    }
    put(p.dscale, col, wp * g1 + bp * g0);
    put(p.dw_post, col, s * g1);
    put(p.db_post, col, s * g0);
}

constexpr int kSms = 148;

template <typename T, int THREADS, int LPR, int NCH>
cudaError_t run_forward(const FhResidualNormParams& p, cudaStream_t st) {
    constexpr int RPC = THREADS / LPR;
    const long long want = (p.m + RPC - 1) / RPC;
    const int grid = (int)std::min<long long>(want, (long long)kSms * 2048 / THREADS);
    return fhk::launch(k_residual_norm<T, THREADS, LPR, NCH>, dim3(grid), dim3(THREADS), 0, st, p,
                       p.gate ? p.m / p.gates : p.m);
}

template <typename T>
cudaError_t forward(const FhResidualNormParams& p, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    if (c8 <= 8) return run_forward<T, 256, 8, 1>(p, st);
    if (c8 <= 32) return run_forward<T, 256, 32, 1>(p, st);
    if (c8 <= 64) return run_forward<T, 256, 32, 2>(p, st);
    if (c8 <= 256) return run_forward<T, 128, 128, 2>(p, st);
    if (c8 <= 512) return run_forward<T, 256, 256, 2>(p, st);
    return run_forward<T, 512, 512, 2>(p, st);
}

Split split_of(long long m, int c, int gates, bool gate) {
    Split s{};
    s.groups = gate ? gates : 1;
    s.len = m / s.groups;
    const int target = c > 2048 ? kSms : 2 * kSms;
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

template <typename T, int THREADS, int LPR, int NCH>
cudaError_t run_grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    return fhk::launch(k_residual_norm_grad<T, THREADS, LPR, NCH>, dim3(sp.ctas), dim3(THREADS), 0, st, p, sp,
                       static_cast<float*>(p.scratch));
}

template <typename T>
cudaError_t grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    cudaError_t e;
    if (c8 <= 8) e = run_grad<T, 256, 8, 1>(p, sp, st);
    else if (c8 <= 32) e = run_grad<T, 256, 32, 1>(p, sp, st);
    else if (c8 <= 128) e = run_grad<T, 128, 128, 1>(p, sp, st);
    else if (c8 <= 256) e = run_grad<T, 256, 256, 1>(p, sp, st);
    else if (c8 <= 512) e = run_grad<T, 512, 512, 1>(p, sp, st);
    else e = run_grad<T, 512, 512, 2>(p, sp, st);
    if (e != cudaSuccess) return e;
    const bool post = p.f && (p.dgate || p.dscale || p.dw_post || p.db_post), pre = p.dw_pre || p.db_pre;
    if (!post && !pre) return cudaSuccess;
    // blockIdx.y selects the side; the post side's blocks return at once where nothing of it is wanted
    return fhk::launch(k_residual_norm_params<T>, dim3((p.c + 31) / 32, 2), dim3(256), 0, st, p, sp,
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
