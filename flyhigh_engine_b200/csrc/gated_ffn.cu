// The gated feed-forward block (fhk_gated_ffn) and its gradient.
//
//   g = x Wg^T + bg, u = x Wu^T + bu, a = act(g) u, y = a Wd^T + bd
//   da = dy Wd; dg = da u act'(g), du = da act(g); dx = dg Wg + du Wu; dWg = dg^T x, dWu = du^T x, dWd = dy^T a
//
// Every one of these is a product over rows or channels with an elementwise tail, so one warp-specialised kernel
// (k_product) computes them all: operands by tensor copies into swizzled tiles, tcgen05.mma into tensor memory, the tail on
// the accumulators as they are read back. An operand may be K-major or MN-major, so no transposed copy of a weight, of x
// or of a gradient is ever made. A forward call is two launches (gate and up projections with activation and
// product; down projection), a gradient two as well (da with the activation's gradient; dx and all weight gradients as
// jobs of one persistent launch), plus, where they apply, one that joins split sums and two for the biases' column sums.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fh_device.cuh"
#include "fh_kernels.h"
#include "launch.h"
#include "row_ops.cuh"
#include "umma_tile.cuh"

using namespace rows;

namespace {

constexpr int kMaxChannels = 1 << 20;
constexpr int kSms = 148;

__device__ unsigned long long g_ffn_timeouts;

// act(g)
template <int ACT>
__device__ __forceinline__ float act_of(float g) {
    if (ACT == FH_ACT_RELU) return g > 0.0f ? g : 0.0f;
    if (ACT == FH_ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678f));
    // 0.5 (1 + tanh z) = sigmoid(2 z), so the tanh form is g sigmoid(2 sqrt(2 / pi) (g + 0.044715 g^3))
    const float z = ACT == FH_ACT_GELU_TANH ? g * (1.59576912f + 0.07135481f * g * g) : g;
    const float s = __fdividef(1.0f, 1.0f + __expf(-z));
    return ACT == FH_ACT_SIGMOID ? s : g * s;
}
// act(g) and its derivative
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& v, float& dv) {
    if (ACT == FH_ACT_RELU) {
        v = g > 0.0f ? g : 0.0f;
        dv = g > 0.0f ? 1.0f : 0.0f;
    } else if (ACT == FH_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678f));
        v = g * cdf;
        dv = cdf + g * 0.39894228f * __expf(-0.5f * g * g);
    } else {
        const float g2 = g * g;
        const float z = ACT == FH_ACT_GELU_TANH ? g * (1.59576912f + 0.07135481f * g2) : g;
        const float s = __fdividef(1.0f, 1.0f + __expf(-z));
        v = ACT == FH_ACT_SIGMOID ? s : g * s;
        dv = ACT == FH_ACT_SIGMOID ? s * (1.0f - s)
             : ACT == FH_ACT_SILU  ? s * (1.0f + g * (1.0f - s))
                                   : s + v * (1.0f - s) * (1.59576912f + 0.21406443f * g2);
    }
}

enum Tail { PLAIN, GLU, GLU_GRAD };

// One product of a launch: out[m][n] = tail(sum over the terms of A[t] B[t]^T). GLU: A[0] with B[0] (gate) and B[1] (up).
struct alignas(64) Job {
    CUtensorMap a[2], b[2];
    int mn_a, mn_b;                // the operand is MN-major
    int kb[2];                     // 64-deep K blocks of the terms
    int m, n;                      // output extents
    int tiles_m, tiles_n, splits;  // tiles, and the parts of K that different CTAs sum
    int first;                     // its first work item
    void *out, *out1, *out2;       // PLAIN: out; GLU: a, and g, u or NULL; GLU_GRAD: dg, du
    long long pitch;
    const void *bias0, *bias1;  // by column, or NULL
    const void *g, *u;          // GLU_GRAD
    float* part;                // splits > 1: [split][m][n8] sums in place of out
};
constexpr int kJobs = 4;
struct Work {
    Job job[kJobs];
    int jobs, items, bn, stages, act;
    long long limit;
};

constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kStageA = 128 * 128;  // 128 rows of 64 elements
constexpr int kRing = 196608;       // shared memory of the operand ring
constexpr int kMaxStages = 8;
constexpr int kSmem = 1024 + kRing + 256;
constexpr int kGroupM = 8;  // tiles of rows that are walked together, so that their operands stay in L2

struct Item {
    const Job* j;
    int tm, tn, split, k0, k1;
};
__device__ __forceinline__ Item item_of(const Work& w, int i) {
    int n = 0;
    while (n + 1 < w.jobs && i >= w.job[n + 1].first) n++;
    const Job& j = w.job[n];
    i -= j.first;
    const int tiles = j.tiles_m * j.tiles_n;
    Item t;
    t.j = &j;
    t.split = i / tiles;
    i -= t.split * tiles;
    const int per = kGroupM * j.tiles_n, grp = i / per;
    const int rows_ = min(kGroupM, j.tiles_m - grp * kGroupM);
    i -= grp * per;
    t.tm = grp * kGroupM + i % rows_;
    t.tn = i / rows_;
    const int kb = j.kb[0] + j.kb[1];
    t.k0 = (int)((long long)kb * t.split / j.splits);
    t.k1 = (int)((long long)kb * (t.split + 1) / j.splits);
    return t;
}

// 16 values of a row into 16 columns, `valid` of them there; wide: the row's columns begin on 32-byte boundaries
template <typename T>
__device__ __forceinline__ void store16(T* p, int valid, bool wide, const float (&v)[16]) {
    if (valid >= 16) {
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = Elem<T>::from2(v[2 * i], v[2 * i + 1]);
        if (wide) {
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]),
                         "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7])
                         : "memory");
        } else {
            reinterpret_cast<uint4*>(p)[0] = make_uint4(q[0], q[1], q[2], q[3]);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(q[4], q[5], q[6], q[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < valid) p[i] = Elem<T>::from(v[i]);
    }
}
template <typename T>
__device__ __forceinline__ void load16g(const T* p, int valid, float (&v)[16]) {
    if (valid >= 16) {
        float t[8];
        load8(p, 8, t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = t[i];
        load8(p + 8, 8, t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[8 + i] = t[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = i < valid ? Elem<T>::to(p[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void add_bias16(const void* bias, int c, int valid, float (&v)[16]) {
    if (!bias) return;
    float b[16];
    load16g(static_cast<const T*>(bias) + c, valid, b);
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] += b[i];
}

template <int ACT>
__device__ __forceinline__ void glu16(const float (&g)[16], const float (&u)[16], float (&a)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) a[i] = act_of<ACT>(g[i]) * u[i];
}
template <int ACT>
__device__ __forceinline__ void glu_grad16(const float (&da)[16], float (&g)[16], float (&u)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
        float v, dv;
        act_both<ACT>(g[i], v, dv);
        g[i] = da[i] * u[i] * dv;
        u[i] = da[i] * v;
    }
}

// CTAS = 2: a pair of CTAs computes 256 x bn tiles, each CTA holding 128 rows of A, half the columns' rows of B and the
// accumulators of its own rows. Warps 0-7 read the accumulators (two per 32 lanes, each half the columns), warp 8 issues the
// copies, warp 9 (of the pair's first CTA) the matrix instructions. The accumulators are double-buffered: a tile's tail
// runs while the next tile's products do.
template <typename T, int CTAS, int TAIL>
__global__ void __launch_bounds__(kThreads, 1) k_product(const __grid_constant__ Work w) {
    extern __shared__ uint8_t raw[];
    using namespace umma;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
    const int bn = w.bn, nb = bn / CTAS, stages = w.stages;
    const uint32_t stage_bytes = kStageA + nb * 128;
    const uint32_t bars = base + kRing;
    const uint32_t full = bars, empty = bars + 8 * kMaxStages, tfull = bars + 16 * kMaxStages, tempty = tfull + 16,
                   slot = tempty + 16;
    const uint32_t cols = 2 * bn;

    if (warp == 8 && lane == 0) {
        for (int s = 0; s < stages; s++) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            bar_init(tfull + 8 * b, 1);
            bar_init(tempty + 8 * b, kEpiWarps * CTAS);
        }
        bar_init_fence();
    }
    if (warp == 9) tmem_alloc<CTAS>(slot, cols);
    fence_before();
    if (CTAS == 2) cluster_sync();
    else __syncthreads();
    fence_after();
    uint32_t tbase;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tbase) : "r"(slot));
    pdl_wait();
    pdl_trigger();

    const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    bool ok = true;
    if (warp == 8) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 1;  // the ring starts empty
            for (int i = first; ok && i < w.items; i += step) {
                const Item t = item_of(w, i);
                const Job& j = *t.j;
                const int row = t.tm * 128 * CTAS + (int)rank * 128;
                for (int k = t.k0; k < t.k1; k++) {
                    if (!bar_wait(empty + 8 * s, ph, w.limit, &g_ffn_timeouts)) {
                        ok = false;
                        break;
                    }
                    const int term = TAIL != GLU && k >= j.kb[0], kk = (k - (term ? j.kb[0] : 0)) * BK;
                    if (rank == 0) bar_expect(full + 8 * s, CTAS * stage_bytes);
                    const uint32_t bar = CTAS == 2 ? map_rank(full + 8 * s, 0) : full + 8 * s;
                    const uint32_t da = base + s * stage_bytes, db = da + kStageA;
                    const CUtensorMap* ma = &j.a[term];
                    if (j.mn_a) {
                        tensor_load<CTAS>(da, ma, row, kk, bar);
                        tensor_load<CTAS>(da + 8192, ma, row + 64, kk, bar);
                    } else {
                        tensor_load<CTAS>(da, ma, kk, row, bar);
                    }
                    if (TAIL == GLU) {
                        const int c = t.tn * (bn / 2);
                        if (CTAS == 2) {
                            tensor_load<CTAS>(db, &j.b[rank], kk, c, bar);
                        } else {
                            tensor_load<CTAS>(db, &j.b[0], kk, c, bar);
                            tensor_load<CTAS>(db + (bn / 2) * 128, &j.b[1], kk, c, bar);
                        }
                    } else {
                        const int c = t.tn * bn + (int)rank * nb;
                        if (j.mn_b)
                            for (int q = 0; q < nb / 64; q++) tensor_load<CTAS>(db + q * 8192, &j.b[term], c + 64 * q, kk, bar);
                        else
                            tensor_load<CTAS>(db, &j.b[term], kk, c, bar);
                    }
                    if (++s == stages) s = 0, ph ^= 1;
                }
            }
        }
    } else if (warp == 9) {
        if (lane == 0 && rank == 0) {
            int s = 0, n = 0;
            uint32_t ph = 0;
            for (int i = first; ok && i < w.items; i += step, n++) {
                const Item t = item_of(w, i);
                const Job& j = *t.j;
                const int b = n & 1;
                const uint32_t d = tbase + b * bn;
                const uint32_t idesc = instr_desc(sizeof(T) == 2 && !std::is_same<T, __half>::value, j.mn_a, j.mn_b, 128 * CTAS, bn);
                // one K step of 16: 32 bytes along a K-major tile's rows, two 8-k groups of an MN-major one
                const uint32_t sa = j.mn_a ? 2048 >> 4 : 32 >> 4, sb = j.mn_b ? 2048 >> 4 : 32 >> 4;
                if (!bar_wait(tempty + 8 * b, ((n >> 1) & 1) ^ 1, w.limit, &g_ffn_timeouts)) {
                    ok = false;
                    break;
                }
                fence_after();
                for (int k = t.k0; k < t.k1; k++) {
                    if (!bar_wait(full + 8 * s, ph, w.limit, &g_ffn_timeouts)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    const uint32_t da = base + s * stage_bytes;
                    const uint64_t ad = tile_desc(da, 8192), bd = tile_desc(da + kStageA, 8192);
#pragma unroll
                    for (int q = 0; q < 4; q++) mma<CTAS>(d, ad + q * sa, bd + q * sb, idesc, (k > t.k0 || q > 0) ? 1u : 0u);
                    commit<CTAS>(empty + 8 * s);
                    if (++s == stages) s = 0, ph ^= 1;
                }
                if (ok) commit<CTAS>(tfull + 8 * b);
            }
        }
    } else {
        const int q = warp & 3, half = warp >> 2;
        int n = 0;
        for (int i = first; i < w.items; i += step, n++) {
            const Item t = item_of(w, i);
            const Job& j = *t.j;
            const int b = n & 1;
            const long long row = (long long)t.tm * 128 * CTAS + rank * 128 + q * 32 + lane;
            const bool on = row < j.m;
            ok = bar_wait(tfull + 8 * b, (n >> 1) & 1, w.limit, &g_ffn_timeouts);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
            const uint32_t acc = tbase + ((uint32_t)(q * 32) << 16) + b * bn;
            if (TAIL == GLU) {
                const bool wide = (j.pitch & 15) == 0 && (((uintptr_t)j.out | (uintptr_t)j.out1 | (uintptr_t)j.out2) & 31) == 0;
                for (int c0 = half * (bn / 4); c0 < (half + 1) * (bn / 4); c0 += 16) {
                    uint32_t rg[16], ru[16];
                    load16(acc + c0, rg);
                    load16(acc + bn / 2 + c0, ru);
                    wait_ld();
                    const int c = t.tn * (bn / 2) + c0, valid = min(16, j.n - c);
                    if (on && valid > 0) {
                        float g[16], u[16], a[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) g[e] = __uint_as_float(rg[e]), u[e] = __uint_as_float(ru[e]);
                        add_bias16<T>(j.bias0, c, valid, g);
                        add_bias16<T>(j.bias1, c, valid, u);
                        switch (w.act) {
                            case FH_ACT_SILU: glu16<FH_ACT_SILU>(g, u, a); break;
                            case FH_ACT_GELU: glu16<FH_ACT_GELU>(g, u, a); break;
                            case FH_ACT_GELU_TANH: glu16<FH_ACT_GELU_TANH>(g, u, a); break;
                            case FH_ACT_RELU: glu16<FH_ACT_RELU>(g, u, a); break;
                            default: glu16<FH_ACT_SIGMOID>(g, u, a); break;
                        }
                        const long long at = row * j.pitch + c;
                        store16(static_cast<T*>(j.out) + at, valid, wide, a);
                        if (j.out1) {
                            store16(static_cast<T*>(j.out1) + at, valid, wide, g);
                            store16(static_cast<T*>(j.out2) + at, valid, wide, u);
                        }
                    }
                    __syncwarp();
                }
            } else {
                const bool wide = (j.pitch & 15) == 0 && (((uintptr_t)j.out | (uintptr_t)j.out1) & 31) == 0;
                for (int c0 = half * (bn / 2); c0 < (half + 1) * (bn / 2); c0 += 16) {
                    const int c = t.tn * bn + c0, valid = min(16, j.n - c);
                    const long long at = row * j.pitch + c;
                    float g[16], u[16];
                    if (TAIL == GLU_GRAD && on && valid > 0) {
                        load16g(static_cast<const T*>(j.g) + at, valid, g);
                        load16g(static_cast<const T*>(j.u) + at, valid, u);
                    }
                    __syncwarp();
                    uint32_t r[16];
                    load16(acc + c0, r);
                    wait_ld();
                    if (on && valid > 0) {
                        float v[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] = __uint_as_float(r[e]);
                        if (TAIL == GLU_GRAD) {
                            switch (w.act) {
                                case FH_ACT_SILU: glu_grad16<FH_ACT_SILU>(v, g, u); break;
                                case FH_ACT_GELU: glu_grad16<FH_ACT_GELU>(v, g, u); break;
                                case FH_ACT_GELU_TANH: glu_grad16<FH_ACT_GELU_TANH>(v, g, u); break;
                                case FH_ACT_RELU: glu_grad16<FH_ACT_RELU>(v, g, u); break;
                                default: glu_grad16<FH_ACT_SIGMOID>(v, g, u); break;
                            }
                            store16(static_cast<T*>(j.out) + at, valid, wide, g);
                            store16(static_cast<T*>(j.out1) + at, valid, wide, u);
                        } else if (j.part) {
                            const long long n8 = (j.n + 7) & ~7;
                            float4* p = reinterpret_cast<float4*>(j.part + ((long long)t.split * j.m + row) * n8 + c);
#pragma unroll
                            for (int e = 0; e < 4; e++)  // columns up to n8 are the scratch's own
                                if (4 * e < valid) p[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                        } else {
                            add_bias16<T>(j.bias0, c, valid, v);
                            store16(static_cast<T*>(j.out) + at, valid, wide, v);
                        }
                    }
                    __syncwarp();
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(CTAS == 2 ? map_rank(tempty + 8 * b, 0) : map_rank(tempty + 8 * b, rank));
        }
    }
    // a role that gave up leaves copies and matrix instructions in flight: give them time before the memory is let go
    if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
    }
    __syncwarp();
    fence_before();
    if (CTAS == 2) cluster_sync();
    else __syncthreads();
    fence_after();
    if (warp == 9) tmem_free<CTAS>(tbase, cols);
}

// The split sums of a launch's jobs added in order, with the bias: 8 columns per thread
struct Join {
    const float* part;
    void* out;
    const void* bias;
    long long pitch, m;
    int n, splits;
    long long first;  // its first group of 8 columns
};
struct Joins {
    Join j[kJobs];
    int n;
    long long total;
};
template <typename T>
__global__ void __launch_bounds__(256) k_join(const Joins w) {
    pdl_wait();
    long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= w.total) return;
    int k = 0;
    while (k + 1 < w.n && i >= w.j[k + 1].first) k++;
    const Join& j = w.j[k];
    i -= j.first;
    const int n8 = (j.n + 7) / 8;
    const long long row = i / n8;
    const int c = (int)(i - row * n8) * 8, valid = min(8, j.n - c);
    float v[8] = {};
    const float* p = j.part + (row * n8 * 8 + c);
    for (int s = 0; s < j.splits; s++, p += j.m * n8 * 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    }
    if (j.bias) {
        float b[8];
        load8(static_cast<const T*>(j.bias) + c, valid, b);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += b[e];
    }
    store8(static_cast<T*>(j.out) + row * j.pitch + c, valid, v);
}

// Column sums of up to three matrices: a CTA sums a slice of the rows of 64 columns (8 threads of 8 columns by 32 rows),
// a second kernel the slices in order
struct Columns {
    const void* x;
    void* out;
    long long pitch;
    int n;
    long long part;  // its first float of the partial sums
};
struct ColumnSums {
    Columns c[3];
    long long m;
    int slices;
    float* part;
};
template <typename T>
__global__ void __launch_bounds__(256) k_column_parts(const ColumnSums w) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s[32][65];
    const Columns& q = w.c[blockIdx.z];
    const int c = blockIdx.x * 64 + 8 * (threadIdx.x & 7), r = threadIdx.x >> 3;
    if (blockIdx.x * 64 >= q.n) return;
    const int valid = max(0, min(8, q.n - c));
    const long long lo = w.m * blockIdx.y / w.slices, hi = w.m * (blockIdx.y + 1) / w.slices;
    float v[8] = {};
    if (valid)
#pragma unroll 4
        for (long long i = lo + r; i < hi; i += 32) {
            float t[8];
            load8(static_cast<const T*>(q.x) + i * q.pitch + c, valid, t);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += t[e];
        }
#pragma unroll
    for (int e = 0; e < 8; e++) s[r][8 * (threadIdx.x & 7) + e] = v[e];
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < q.n) {
        float t = 0.0f;
        for (int i = 0; i < 32; i++) t += s[i][threadIdx.x];
        w.part[q.part + (long long)blockIdx.y * q.n + blockIdx.x * 64 + threadIdx.x] = t;
    }
}
template <typename T>
__global__ void __launch_bounds__(128) k_column_join(const ColumnSums w) {
    pdl_wait();
    const Columns& q = w.c[blockIdx.y];
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= q.n) return;
    float t = 0.0f;
    for (int i = 0; i < w.slices; i++) t += w.part[q.part + (long long)i * q.n + c];
    static_cast<T*>(q.out)[c] = Elem<T>::from(t);
}

#define FH_TRY(call)                              \
    do {                                          \
        const cudaError_t e_ = (call);            \
        if (e_ != cudaSuccess) return e_;         \
    } while (0)

// ---- host: tensor maps, the choice of tiles, launches ----

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

// boxes of 64 columns x `box` rows
cudaError_t map_of(CUtensorMap* map, const Matrix& x, int box, int dtype) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)x.cols, (cuuint64_t)x.rows}, strides[1] = {(cuuint64_t)x.pitch * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, one[2] = {1, 1};
    const CUresult r = fn(map, dtype == FH_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                          const_cast<void*>(x.p), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// A product before its tiles are chosen: terms of (A, B) with A [m][k] (or [k][m], mn_a) and B [n][k] (or [k][n], mn_b)
struct Product {
    Matrix a[2], b[2];
    int terms;
    bool mn_a, mn_b;
    long long m;
    int n;
    long long k;  // of each term
    bool can_split;
    void *out, *out1, *out2;
    long long pitch;
    const void *bias0, *bias1, *g, *u;
};

struct Shape {
    int ctas, bn, splits[kJobs];
};

// The tiles of a launch: 256 x 256 or 256 x 128 by a pair of CTAs, or 128 x 128 or 128 x 64 by one; and into how many
// parts K is cut where the tiles leave SMs idle. Chosen by an estimate in SM cycles: a K block of 64 takes the larger of the
// matrix pipe (128 x bn x 16 in bn / 2 cycles, 46 at least) and its operands' way into shared memory (about 56 bytes per
// cycle and SM), a CTA runs ceil(items / slots) tiles one after another, each followed by a tail that the next tile's products
// hide, and split sums are written, read and joined by another launch.
template <int TAIL>
Shape shape_of(const Product* p, int n) {
    static const int kinds[4][2] = {{2, 256}, {2, 128}, {1, 128}, {1, 64}};
    Shape best{};
    double best_t = 1e300;
    for (const auto& kind : kinds) {
        Shape s{};
        s.ctas = kind[0], s.bn = kind[1];
        const int slots = kSms / s.ctas, cols = TAIL == GLU ? s.bn / 2 : s.bn;
        const double per_kb = std::max({2.0 * s.bn, 184.0, (128.0 + s.bn / s.ctas) * 128 / 56});
        const double tail = 600.0 + s.bn * (TAIL == PLAIN ? 3.0 : TAIL == GLU ? 5.0 : 9.0);
        double busy = 0, longest = 0, extra = 0;
        bool split_any = false;
        for (int i = 0; i < n; i++) {
            const double tiles = (double)((p[i].m + 128 * s.ctas - 1) / (128 * s.ctas)) * ((p[i].n + cols - 1) / cols);
            const long long kb = (p[i].k + 63) / 64 * p[i].terms;
            int sp = 1;
            if (p[i].can_split && tiles < slots / 2) {
                sp = (int)std::min<double>(std::min<double>(slots / tiles, kb / 4), 64);
                if (sp < 2) sp = 1;
            }
            s.splits[i] = sp;
            const double item = std::max((double)((kb + sp - 1) / sp) * per_kb, tail);
            busy += tiles * sp * item;
            longest = std::max(longest, item);
            if (sp > 1) {
                split_any = true;
                extra += (double)p[i].m * p[i].n * (sp + 0.5) * 4 / 3000;
            }
        }
        const double t = std::max(longest, std::ceil(busy / slots / longest - 1e-9) * longest) + tail + (split_any ? 5000 : 0) + extra;
        if (t < best_t) best_t = t, best = s;
    }
    return best;
}

size_t part_floats(const Product& p, int splits) {
    return splits > 1 ? (size_t)splits * (size_t)p.m * (size_t)((p.n + 7) & ~7) : 0;
}
template <int TAIL>
size_t scratch_floats(const Product* p, int n) {
    const Shape s = shape_of<TAIL>(p, n);
    size_t f = 0;
    for (int i = 0; i < n; i++) f += part_floats(p[i], s.splits[i]);
    return f;
}

template <typename T, int CTAS, int TAIL>
cudaError_t launch_work(const Work& w, cudaStream_t st) {
    static std::atomic<bool> prepared[64];  // per device
    int dev = 0;
    FH_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!prepared[dev].load(std::memory_order_acquire)) {
        FH_TRY(cudaFuncSetAttribute(k_product<T, CTAS, TAIL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        prepared[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min(w.items, kSms / CTAS) * CTAS);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    unsigned na = 0;
    if (CTAS == 2) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim = {2, 1, 1};
        na++;
    }
    if (fhk::pdl_flag()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    return cudaLaunchKernelEx(&cfg, k_product<T, CTAS, TAIL>, w);
}

// the products of one launch (and the launch that joins their split sums); part: scratch_floats
template <typename T, int TAIL>
cudaError_t products(const Product* p, int n, int act, int dtype, long long limit, float* part, cudaStream_t st) {
    const Shape s = shape_of<TAIL>(p, n);
    Work w;
    w.jobs = n, w.items = 0, w.bn = s.bn, w.act = act, w.limit = limit > 0 ? limit : 2000000000ll;
    const int nb = s.bn / s.ctas;
    w.stages = std::min(kMaxStages, kRing / (kStageA + nb * 128));
    Joins joins{};
    for (int i = 0; i < n; i++) {
        Job& j = w.job[i];
        const Product& q = p[i];
        for (int t = 0; t < (TAIL == GLU ? 2 : q.terms); t++) {
            if (t == 0 || TAIL != GLU) FH_TRY(map_of(&j.a[t], q.a[t], q.mn_a ? 64 : 128, dtype));
            FH_TRY(map_of(&j.b[t], q.b[t], q.mn_b ? 64 : TAIL == GLU ? s.bn / 2 : nb, dtype));
        }
        const int kb = (int)((q.k + 63) / 64);
        j.mn_a = q.mn_a, j.mn_b = q.mn_b, j.kb[0] = kb, j.kb[1] = q.terms > 1 ? kb : 0, j.m = (int)q.m, j.n = q.n;
        j.tiles_m = (int)((q.m + 128 * s.ctas - 1) / (128 * s.ctas));
        const int cols = TAIL == GLU ? s.bn / 2 : s.bn;
        j.tiles_n = (q.n + cols - 1) / cols;
        j.splits = s.splits[i];
        j.first = w.items;
        const long long items = w.items + (long long)j.tiles_m * j.tiles_n * j.splits;
        if (items > (1ll << 30)) return cudaErrorInvalidValue;
        w.items = (int)items;
        j.out = q.out, j.out1 = q.out1, j.out2 = q.out2, j.pitch = q.pitch, j.bias0 = q.bias0, j.bias1 = q.bias1, j.g = q.g, j.u = q.u;
        j.part = nullptr;
        if (j.splits > 1) {
            j.part = part;
            Join& o = joins.j[joins.n++];
            o = {part, q.out, q.bias0, q.pitch, q.m, q.n, j.splits, joins.total};
            joins.total += q.m * ((q.n + 7) / 8);
            part += part_floats(q, j.splits);
        }
    }
    FH_TRY((s.ctas == 2 ? launch_work<T, 2, TAIL>(w, st) : launch_work<T, 1, TAIL>(w, st)));
    if (joins.n) FH_TRY(fhk::launch(k_join<T>, dim3((unsigned)((joins.total + 255) / 256)), dim3(256), 0, st, joins));
    return cudaSuccess;
}

template <typename P>
bool good_sizes(const P* p) {
    return p->m >= 0 && p->m <= kMaxRows && p->cin >= 1 && p->cin <= kMaxChannels && p->hidden >= 1 &&
           p->hidden <= kMaxChannels && p->cout >= 1 && p->cout <= kMaxChannels && p->act >= FH_ACT_SILU &&
           p->act <= FH_ACT_SIGMOID && (p->dtype == FH_F16 || p->dtype == FH_BF16) && p->wait_cycles >= 0;
}
template <typename P>
bool good_weights(const P* p) {
    return good_rows(p->w_gate, p->wg_pitch, p->cin, p->hidden) && good_rows(p->w_up, p->wu_pitch, p->cin, p->hidden) &&
           good_rows(p->w_down, p->wd_pitch, p->hidden, p->cout);
}


Product glu_of(const FhGatedFfnParams& p) {
    Product q{};
    q.a[0] = {p.x, p.x_pitch, p.m, p.cin};
    q.b[0] = {p.w_gate, p.wg_pitch, p.hidden, p.cin};
    q.b[1] = {p.w_up, p.wu_pitch, p.hidden, p.cin};
    q.terms = 1, q.m = p.m, q.n = p.hidden, q.k = p.cin;
    q.out = p.a, q.out1 = p.g, q.out2 = p.u, q.pitch = p.h_pitch, q.bias0 = p.b_gate, q.bias1 = p.b_up;
    return q;
}
Product down_of(const FhGatedFfnParams& p) {
    Product q{};
    q.a[0] = {p.a, p.h_pitch, p.m, p.hidden};
    q.b[0] = {p.w_down, p.wd_pitch, p.cout, p.hidden};
    q.terms = 1, q.m = p.m, q.n = p.cout, q.k = p.hidden, q.can_split = true;
    q.out = p.y, q.pitch = p.y_pitch, q.bias0 = p.b_down;
    return q;
}

template <typename T>
cudaError_t forward(const FhGatedFfnParams& p, cudaStream_t st) {
    const Product glu = glu_of(p), down = down_of(p);
    FH_TRY((products<T, GLU>(&glu, 1, p.act, p.dtype, p.wait_cycles, nullptr, st)));
    fhk::PdlScope pdl(true);  // what follows waits on a kernel of this file
    return products<T, PLAIN>(&down, 1, p.act, p.dtype, p.wait_cycles, static_cast<float*>(p.scratch), st);
}

// the gradient's scratch: dg and du [m][h_pitch], then the split sums and the partial column sums
struct GradPlan {
    Product da, out[kJobs];
    int outs;
    size_t hidden_bytes, part_bytes, column_bytes;
    ColumnSums cols;
    int ncols, widest;
};
GradPlan grad_plan(const FhGatedFfnGradParams& p) {
    GradPlan g{};
    g.hidden_bytes = ((size_t)p.m * p.h_pitch * 2 + 255) / 256 * 256;
    char* dg = static_cast<char*>(p.scratch);
    char* du = dg + g.hidden_bytes;
    g.da.a[0] = {p.dy, p.dy_pitch, p.m, p.cout};
    g.da.b[0] = {p.w_down, p.wd_pitch, p.cout, p.hidden};
    g.da.mn_b = true;
    g.da.terms = 1, g.da.m = p.m, g.da.n = p.hidden, g.da.k = p.cout;
    g.da.out = dg, g.da.out1 = du, g.da.pitch = p.h_pitch, g.da.g = p.g, g.da.u = p.u;
    if (p.dx) {
        Product& q = g.out[g.outs++];
        q.a[0] = {dg, p.h_pitch, p.m, p.hidden};
        q.a[1] = {du, p.h_pitch, p.m, p.hidden};
        q.b[0] = {p.w_gate, p.wg_pitch, p.hidden, p.cin};
        q.b[1] = {p.w_up, p.wu_pitch, p.hidden, p.cin};
        q.mn_b = true;
        q.terms = 2, q.m = p.m, q.n = p.cin, q.k = p.hidden, q.can_split = true, q.out = p.dx, q.pitch = p.dx_pitch;
    }
    auto weight = [&](Matrix left, Matrix right, void* out, long long pitch) {
        if (!out) return;
        Product& q = g.out[g.outs++];
        q.a[0] = left, q.b[0] = right, q.mn_a = q.mn_b = true;
        q.terms = 1, q.m = left.cols, q.n = right.cols, q.k = p.m, q.can_split = true, q.out = out, q.pitch = pitch;
    };
    const Matrix x = {p.x, p.x_pitch, p.m, p.cin};
    weight({dg, p.h_pitch, p.m, p.hidden}, x, p.dw_gate, p.dwg_pitch);
    weight({du, p.h_pitch, p.m, p.hidden}, x, p.dw_up, p.dwu_pitch);
    weight({p.dy, p.dy_pitch, p.m, p.cout}, {p.a, p.h_pitch, p.m, p.hidden}, p.dw_down, p.dwd_pitch);
    g.part_bytes = (g.outs ? scratch_floats<PLAIN>(g.out, g.outs) * 4 + 255 : 0) / 256 * 256;
    auto column = [&](const void* x_, long long pitch, int n, void* out) {
        if (!out) return;
        g.cols.c[g.ncols++] = {x_, out, pitch, n, (long long)g.column_bytes};
        g.column_bytes += n;
        g.widest = std::max(g.widest, n);
    };
    column(dg, p.h_pitch, p.hidden, p.db_gate);
    column(du, p.h_pitch, p.hidden, p.db_up);
    column(p.dy, p.dy_pitch, p.cout, p.db_down);
    if (g.ncols) {
        // about four CTAs per SM over the columns, 64 rows to a slice at least
        const long long across = (long long)((g.widest + 63) / 64) * g.ncols;
        g.cols.slices = (int)std::max<long long>(1, std::min<long long>(std::min<long long>((p.m + 63) / 64, 4 * kSms / across), 1024));
        for (int i = 0; i < g.ncols; i++) g.cols.c[i].part *= g.cols.slices;
        g.column_bytes *= (size_t)g.cols.slices * 4;
        g.cols.m = p.m;
        g.cols.part = reinterpret_cast<float*>(dg + 2 * g.hidden_bytes + g.part_bytes);
    }
    return g;
}

template <typename T>
cudaError_t gradient(const FhGatedFfnGradParams& p, cudaStream_t st) {
    const GradPlan g = grad_plan(p);
    const bool hidden = p.dx || p.dw_gate || p.dw_up || p.db_gate || p.db_up;  // whether dg or du is read
    if (hidden) FH_TRY((products<T, GLU_GRAD>(&g.da, 1, p.act, p.dtype, p.wait_cycles, nullptr, st)));
    fhk::PdlScope pdl(hidden);
    if (g.outs)
        FH_TRY((products<T, PLAIN>(g.out, g.outs, p.act, p.dtype, p.wait_cycles,
                                   reinterpret_cast<float*>(static_cast<char*>(p.scratch) + 2 * g.hidden_bytes), st)));
    if (g.ncols) {
        FH_TRY(fhk::launch(k_column_parts<T>, dim3((g.widest + 63) / 64, g.cols.slices, g.ncols), dim3(256), 0, st, g.cols));
        fhk::PdlScope own(true);
        FH_TRY(fhk::launch(k_column_join<T>, dim3((g.widest + 127) / 128, g.ncols), dim3(128), 0, st, g.cols));
    }
    return cudaSuccess;
}

}  // namespace

extern "C" size_t fhk_gated_ffn_scratch_bytes(const FhGatedFfnParams* p) {
    if (!p || !good_sizes(p) || p->m == 0) return 0;
    const Product down = down_of(*p);
    return scratch_floats<PLAIN>(&down, 1) * 4;
}

extern "C" int fhk_gated_ffn(const FhGatedFfnParams* p, void* stream) {
    if (!p || !good_sizes(p) || !good_weights(p)) return (int)cudaErrorInvalidValue;
    if (!aligned16(p->b_gate) || !aligned16(p->b_up) || !aligned16(p->b_down)) return (int)cudaErrorInvalidValue;
    if (!good_rows(p->x, p->x_pitch, p->cin, p->m) || !good_rows(p->y, p->y_pitch, p->cout, p->m) ||
        !good_rows(p->a, p->h_pitch, p->hidden, p->m) || (p->g != nullptr) != (p->u != nullptr) ||
        !good_rows_or_null(p->g, p->h_pitch, p->hidden, p->m) || !good_rows_or_null(p->u, p->h_pitch, p->hidden, p->m))
        return (int)cudaErrorInvalidValue;
    const size_t need = fhk_gated_ffn_scratch_bytes(p);
    if (need && (!p->scratch || !aligned16(p->scratch) || p->scratch_bytes < need)) return (int)cudaErrorInvalidValue;
    if (p->m == 0) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return (int)(p->dtype == FH_F16 ? forward<__half>(*p, st) : forward<__nv_bfloat16>(*p, st));
}

extern "C" size_t fhk_gated_ffn_grad_scratch_bytes(const FhGatedFfnGradParams* p) {
    if (!p || !good_sizes(p) || p->m == 0 || p->h_pitch <= 0) return 0;
    const GradPlan g = grad_plan(*p);
    return 2 * g.hidden_bytes + g.part_bytes + g.column_bytes;
}

extern "C" int fhk_gated_ffn_grad(const FhGatedFfnGradParams* p, void* stream) {
    if (!p || !good_sizes(p) || !good_weights(p)) return (int)cudaErrorInvalidValue;
    if (!good_rows(p->x, p->x_pitch, p->cin, p->m) || !good_rows(p->dy, p->dy_pitch, p->cout, p->m) ||
        !good_rows(p->g, p->h_pitch, p->hidden, p->m) || !good_rows(p->u, p->h_pitch, p->hidden, p->m) ||
        !good_rows(p->a, p->h_pitch, p->hidden, p->m) || !good_rows_or_null(p->dx, p->dx_pitch, p->cin, p->m) ||
        !good_rows_or_null(p->dw_gate, p->dwg_pitch, p->cin, p->hidden) ||
        !good_rows_or_null(p->dw_up, p->dwu_pitch, p->cin, p->hidden) ||
        !good_rows_or_null(p->dw_down, p->dwd_pitch, p->hidden, p->cout))
        return (int)cudaErrorInvalidValue;
    if (!aligned16(p->db_gate) || !aligned16(p->db_up) || !aligned16(p->db_down)) return (int)cudaErrorInvalidValue;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->m == 0) {  // no rows: the gradients of what all rows share are zero
        auto zero = [&](void* v, long long pitch, int c, int n) {
            return v ? cudaMemset2DAsync(v, 2 * (size_t)pitch, 0, 2 * (size_t)c, (size_t)n, st) : cudaSuccess;
        };
        cudaError_t e = zero(p->dw_gate, p->dwg_pitch, p->cin, p->hidden);
        if (e == cudaSuccess) e = zero(p->dw_up, p->dwu_pitch, p->cin, p->hidden);
        if (e == cudaSuccess) e = zero(p->dw_down, p->dwd_pitch, p->hidden, p->cout);
        if (e == cudaSuccess) e = zero(p->db_gate, p->hidden, p->hidden, 1);
        if (e == cudaSuccess) e = zero(p->db_up, p->hidden, p->hidden, 1);
        if (e == cudaSuccess) e = zero(p->db_down, p->cout, p->cout, 1);
        return (int)e;
    }
    const size_t need = fhk_gated_ffn_grad_scratch_bytes(p);
    if (!p->scratch || !aligned16(p->scratch) || p->scratch_bytes < need) return (int)cudaErrorInvalidValue;
    return (int)(p->dtype == FH_F16 ? gradient<__half>(*p, st) : gradient<__nv_bfloat16>(*p, st));
}

extern "C" long long fhk_gated_ffn_wait_timeouts(int reset) {
    unsigned long long n = 0;
    if (cudaMemcpyFromSymbol(&n, g_ffn_timeouts, sizeof(n)) != cudaSuccess) return -1;
    if (reset) {
        const unsigned long long z = 0;
        if (cudaMemcpyToSymbol(g_ffn_timeouts, &z, sizeof(z)) != cudaSuccess) return -1;
    }
    return (long long)n;
}
